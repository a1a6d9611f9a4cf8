// kivi_pages.cu -- writing new tokens into the paged store and reading them back.
//
// Streaming: a row is read once and written once.  What bounds it is instruction issue
// (a row of codes costs a range, a division and a reciprocal, and five packed
// instructions a pair): 16 x 2048 bf16 tokens of 8 x 128 into 8-bit pages take 81 us
// (150 MB of DRAM traffic, issue slots 75% busy), their read-back 38 us (145 MB, 3.8 TB/s,
// 72%); eight ragged sequences of up to 8192 tokens are read back in 50 us (5.6 TB/s).
#include <math.h>

#include <algorithm>

#include "kivi_internal.cuh"
#include "kivi_pages.cuh"

namespace kivi {
namespace {

template <int T> struct Elem;
template <> struct Elem<kF32> { using type = float; };
template <> struct Elem<kF16> { using type = __half; };
template <> struct Elem<kBF16> { using type = __nv_bfloat16; };
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class E> __device__ __forceinline__ E from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
    return __float2bfloat16_rn(x);
}

// The sequence that owns dense row `tok`: the last i with cu[i] <= tok, found by
// the whole warp, 32 probes a step.
__device__ __forceinline__ int find_sequence(const PagesBatch &b, int tok) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = b.batch;
    while (n > 1) {
        const int step = (n + 31) / 32;
        const int i = (lane + 1) * step;
        const bool below = i < n && __ldg(b.cu + lo + i) <= tok;
        const int c = __popc(__ballot_sync(0xffffffffu, below));
        lo += c * step;
        n = min(step, n - c * step);
    }
    return lo;
}

// Eight consecutive elements to p.
template <class E> __device__ __forceinline__ void store8(E *p, bool vec, const float (&x)[8]) {
    if (vec) {
        constexpr int W = sizeof(E) / 2;
        uint4 w[W];
        E *e = reinterpret_cast<E *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f<E>(x[i]);
#pragma unroll
        for (int i = 0; i < W; ++i) __stcs(reinterpret_cast<uint4 *>(p) + i, w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = from_f<E>(x[i]);
    }
}

// 16 bytes of elements at p (8 of 16 bits, or one word of W for fp32), as loaded.
template <class E> struct Raw {
    static constexpr int W = sizeof(E) / 2;
    uint4 w[W];
    __device__ __forceinline__ void load(const E *p, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < W; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
        } else {
            E *e = reinterpret_cast<E *>(w);
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = p[i];
        }
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const {
        const E *e = reinterpret_cast<const E *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(e[i]);
    }
};

// How a launch divides its work.  One row of D elements belongs to L = D / 8 rounded
// up to a power of two lanes, eight elements each, so a warp step takes R = 32 / L of
// a token's 2 H rows (keys' heads, then values').  A token is 2^log_parts warps',
// which take its steps in turn: one warp where there are tokens enough, since finding
// a token's sequence and page costs as much as a step; a warp for each step where
// there are few and latency counts.
struct Work {
    int L, R, steps, log_parts;
};
constexpr int kAhead = 2; // steps whose loads are in flight at once
constexpr int kSms = 148; // of a B200

// The token of this warp: its slot in the store, or false where it has none.
struct Place {
    int64_t row0; // row number of its slot in head 0's block
    bool there;
};
__device__ __forceinline__ Place find_place(const PagesStore &st, const PagesBatch &b, int tok, bool &owned) {
    const int i = find_sequence(b, tok);
    const Span s = pages_span(b, st, i);
    const int at = tok - s.start, t = s.kv - s.n + at;
    owned = at >= 0 && at < s.n;
    Place p{0, false};
    if (!owned || t < 0) return p;
    const int page = pages_page(b, st, i, t);
    p.there = page >= 0;
    p.row0 = pages_row(st, max(page, 0), 0, t);
    return p;
}

__device__ __forceinline__ float min3f(float a, float b, float c) {
    float d;
    asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// clamp(rint((x - zero) / scale), 0, levels) by an IEEE quotient, in the low bits
__device__ __noinline__ uint32_t exact_code(float x, float zero, float scale, float levels) {
    float q = scale == 0.0f ? 0.0f : rintf(__fdiv_rn(__fsub_rn(x, zero), scale));
    q = fminf(fmaxf(q, 0.0f), levels);
    return __float_as_uint(__fadd_rn(q, 8388608.0f));
}

// Eight codes of a row with (scale, zero), packed: exact_code of each.  With d = x -
// zero, fma(d, 1 / scale, 2^23) rounds the exact product d * rcp half to even into the
// low mantissa bits, and e is that product's distance from the integer; product and
// quotient differ by less than 2^(BITS-23), so where |e| <= 1/2 - 2^(BITS-22) both round
// to the same integer, which lies in 0 .. levels.  The others (near ties, which 0.4% of
// bf16 values are: their differences and spans have few bits; NaN; a scale without a
// normal reciprocal) are divided one by one.
template <int BITS>
__device__ __forceinline__ void pack8(const float (&x)[8], float zero, float scale, uint32_t &lo, uint32_t &hi) {
    constexpr float levels = (float)((1 << BITS) - 1), magic = 8388608.0f;
    const bool fast = scale >= 0x1p-125f && scale <= 0x1p125f;
    const float limit = fast ? 0.5f - (float)(1u << BITS) * 0x1p-22f : -1.0f, rcp = fast ? __frcp_rn(scale) : 0.0f;
    uint32_t c[8];
    float e[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2 d = __fadd2_rn(make_float2(x[j], x[j + 1]), make_float2(-zero, -zero));
        const float2 r2 = make_float2(rcp, rcp), m2 = make_float2(magic, magic);
        const float2 rm = __ffma2_rn(d, r2, m2);
        const float2 nr = __ffma2_rn(rm, make_float2(-1.0f, -1.0f), m2); // minus the integer
        const float2 f = __ffma2_rn(d, r2, nr);
        c[j] = __float_as_uint(rm.x), c[j + 1] = __float_as_uint(rm.y);
        e[j] = f.x, e[j + 1] = f.y;
    }
    const float dev = max3_nan(max3_nan(fabsf(e[0]), fabsf(e[1]), fabsf(e[2])), max3_nan(fabsf(e[3]), fabsf(e[4]), fabsf(e[5])),
                               max3_nan(fabsf(e[6]), fabsf(e[7]), fabsf(e[7])));
    if (!(dev <= limit)) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (!(fabsf(e[j]) <= limit)) c[j] = exact_code(x[j], zero, scale, levels);
    }
    if constexpr (BITS == 8) {
        lo = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
        hi = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
    } else {
        // pairs into bytes, then four bytes into the word
        uint32_t p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = (c[2 * j] & 15u) | (c[2 * j + 1] & 15u) << 4;
        lo = __byte_perm(__byte_perm(p[0], p[1], 0x0040), __byte_perm(p[2], p[3], 0x0040), 0x5410);
        hi = 0;
    }
}

// Minimum and maximum of a row, NaN left out, over its L lanes: as (min, -max), so that
// one minimum does for both; 16-bit elements stay packed in a word, which halves the
// shuffles as well.
template <int T> struct Range {
    float mn, nx;
    __device__ __forceinline__ void of(const Raw<float> &r, bool live) {
        float e[8];
        r.floats(e);
        mn = live ? min3f(min3f(e[0], e[1], e[2]), min3f(e[3], e[4], e[5]), fminf(e[6], e[7])) : INFINITY;
        nx = live ? -max3f(max3f(e[0], e[1], e[2]), max3f(e[3], e[4], e[5]), fmaxf(e[6], e[7])) : INFINITY;
    }
    __device__ __forceinline__ void join(int o, bool in) {
        const float a = __shfl_xor_sync(0xffffffffu, mn, o), b = __shfl_xor_sync(0xffffffffu, nx, o);
        if (in) mn = fminf(mn, a), nx = fminf(nx, b);
    }
    __device__ __forceinline__ float least() const { return mn; }
    __device__ __forceinline__ float most() const { return -nx; }
};
template <int T> struct Range16 {
    uint32_t v; // (min, -max)
    __device__ __forceinline__ static uint32_t min2(uint32_t a, uint32_t b) {
        uint32_t d;
        if constexpr (T == kBF16) asm("min.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("min.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    __device__ __forceinline__ static uint32_t max2(uint32_t a, uint32_t b) {
        uint32_t d;
        if constexpr (T == kBF16) asm("max.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        else asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
        return d;
    }
    template <class E> __device__ __forceinline__ void of(const Raw<E> &r, bool live) {
        const uint4 w = r.w[0];
        const uint32_t a = min2(min2(w.x, w.y), min2(w.z, w.w)), b = max2(max2(w.x, w.y), max2(w.z, w.w)) ^ 0x80008000u;
        v = min2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
        if (!live) v = T == kBF16 ? 0x7f807f80u : 0x7c007c00u; // infinities
    }
    __device__ __forceinline__ void join(int o, bool in) {
        const uint32_t a = __shfl_xor_sync(0xffffffffu, v, o);
        if (in) v = min2(v, a);
    }
    __device__ __forceinline__ static float f(uint16_t h) {
        return T == kBF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
    }
    __device__ __forceinline__ float least() const { return f((uint16_t)v); }
    __device__ __forceinline__ float most() const { return -f((uint16_t)(v >> 16)); }
};
template <> struct Range<kBF16> : Range16<kBF16> {};
template <> struct Range<kF16> : Range16<kF16> {};

template <int BITS, int T>
__global__ void __launch_bounds__(256) pages_write_kernel(PagesStore st, PagesBatch b, PagesDense x, Work w) {
    using E = typename Elem<T>::type;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int tok = (int)(id >> w.log_parts), part = (int)id & ((1 << w.log_parts) - 1);
    if (tok >= b.total) return;
    const int sub = lane / w.L, c = lane % w.L * 8;
    const bool in = c < st.D;
    bool owned = false;
    Place at{0, false};
    for (int s0 = part; s0 < w.steps; s0 += kAhead << w.log_parts) {
        Raw<E> raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = (s0 + (u << w.log_parts)) * w.R + sub;
            if (r < 2 * st.H && in) {
                const bool value = r >= st.H;
                raw[u].load(static_cast<const E *>(value ? x.v : x.k) + tok * x.token + (value ? r - st.H : r) * x.head + c, x.vec);
            }
        }
        if (s0 == part) { // while the first loads are under way
            at = find_place(st, b, tok, owned);
            if (!at.there) return; // the whole warp
        }
        Range<T> range[kAhead];
        if constexpr (BITS < 16) { // the steps' reductions side by side
#pragma unroll
            for (int u = 0; u < kAhead; ++u) range[u].of(raw[u], in && (s0 + (u << w.log_parts)) * w.R + sub < 2 * st.H);
            // lanes of another row never mix in: the butterfly stays within L lanes
#pragma unroll
            for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                for (int u = 0; u < kAhead; ++u) range[u].join(o, o < w.L);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = (s0 + (u << w.log_parts)) * w.R + sub;
            if (r >= 2 * st.H || !in) continue;
            const bool value = r >= st.H;
            const int64_t row = at.row0 + ((int64_t)(value ? r - st.H : r) << st.shift);
            unsigned char *dst = (value ? st.v : st.k) + row * st.row_bytes;
            if constexpr (BITS == 16) {
                if constexpr (T != kF32) {
                    if (T == st.dtype) { // as it came
                        *reinterpret_cast<uint4 *>(dst + 2 * c) = raw[u].w[0];
                        continue;
                    }
                }
                float e[8];
                raw[u].floats(e);
                if (st.dtype == kBF16)
                    store8(reinterpret_cast<__nv_bfloat16 *>(dst) + c, true, e);
                else
                    store8(reinterpret_cast<__half *>(dst) + c, true, e);
            } else {
                float e[8];
                raw[u].floats(e);
                const float mn = range[u].least(), span = __fsub_rn(range[u].most(), mn);
                const float scale = span == 0.0f ? 0.0f : __fdiv_rn(span, (float)((1 << BITS) - 1));
                uint32_t lo, hi;
                pack8<BITS>(e, mn, scale, lo, hi);
                if constexpr (BITS == 8)
                    *reinterpret_cast<uint2 *>(dst + c) = make_uint2(lo, hi);
                else
                    *reinterpret_cast<uint32_t *>(dst + c / 2) = lo;
                if (c == 0) (value ? st.vp : st.kp)[row] = make_float2(scale, mn);
            }
        }
        __syncwarp();
    }
}

template <int BITS, int T>
__global__ void __launch_bounds__(256) pages_read_kernel(PagesStore st, PagesBatch b, PagesDense x, Work w) {
    using E = typename Elem<T>::type;
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int tok = (int)(id >> w.log_parts), part = (int)id & ((1 << w.log_parts) - 1);
    if (tok >= b.total) return;
    const int sub = lane / w.L, c = lane % w.L * 8;
    const bool in = c < st.D;
    bool owned;
    const Place at = find_place(st, b, tok, owned);
    if (!owned) return;
    for (int s0 = part; s0 < w.steps; s0 += kAhead << w.log_parts) {
        uint4 raw[kAhead];
        float2 par[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = (s0 + (u << w.log_parts)) * w.R + sub;
            raw[u] = make_uint4(0, 0, 0, 0);
            par[u] = make_float2(0.0f, 0.0f);
            if (r < 2 * st.H && in && at.there) {
                const bool value = r >= st.H;
                const int64_t row = at.row0 + ((int64_t)(value ? r - st.H : r) << st.shift);
                const unsigned char *src = (value ? st.v : st.k) + row * st.row_bytes;
                if constexpr (BITS == 16) {
                    raw[u] = __ldcs(reinterpret_cast<const uint4 *>(src + 2 * c));
                } else {
                    if constexpr (BITS == 8) {
                        const uint2 y = __ldcs(reinterpret_cast<const uint2 *>(src + c));
                        raw[u].x = y.x, raw[u].y = y.y;
                    } else {
                        raw[u].x = __ldcs(reinterpret_cast<const uint32_t *>(src + c / 2));
                    }
                    par[u] = __ldg((value ? st.vp : st.kp) + row);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = (s0 + (u << w.log_parts)) * w.R + sub;
            if (r >= 2 * st.H || !in) continue;
            const bool value = r >= st.H;
            E *dst = static_cast<E *>(const_cast<void *>(value ? x.v : x.k)) + tok * x.token + (value ? r - st.H : r) * x.head + c;
            float e[8];
            if constexpr (BITS == 16) {
                if constexpr (T != kF32) {
                    if (T == st.dtype && x.vec) {
                        __stcs(reinterpret_cast<uint4 *>(dst), raw[u]);
                        continue;
                    }
                }
                const uint32_t v[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint16_t h = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
                    e[j] = st.dtype == kBF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
                }
            } else {
                // the code in the mantissa of 2^23, less 2^23: exact
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    uint32_t a, z;
                    if constexpr (BITS == 8) {
                        a = __byte_perm(j < 4 ? raw[u].x : raw[u].y, 0x4B000000u, 0x7440u | (j & 3));
                        z = __byte_perm(j < 4 ? raw[u].x : raw[u].y, 0x4B000000u, 0x7441u + (j & 3));
                    } else {
                        a = (raw[u].x >> (4 * j) & 15u) | 0x4B000000u, z = (raw[u].x >> (4 * j + 4) & 15u) | 0x4B000000u;
                    }
                    const float2 q = __fadd2_rn(make_float2(__uint_as_float(a), __uint_as_float(z)), make_float2(-8388608.0f, -8388608.0f));
                    const float2 y = __ffma2_rn(q, make_float2(par[u].x, par[u].x), make_float2(par[u].y, par[u].y));
                    e[j] = y.x, e[j + 1] = y.y;
                }
            }
            store8(dst, x.vec, e);
        }
    }
}

template <template <int, int> class F, class... A>
cudaError_t by_type(int bits, int dtype, A &&...a) {
    if (bits == 16)
        return dtype == kF32 ? F<16, kF32>::go(a...) : dtype == kF16 ? F<16, kF16>::go(a...) : F<16, kBF16>::go(a...);
    if (bits == 8)
        return dtype == kF32 ? F<8, kF32>::go(a...) : dtype == kF16 ? F<8, kF16>::go(a...) : F<8, kBF16>::go(a...);
    return dtype == kF32 ? F<4, kF32>::go(a...) : dtype == kF16 ? F<4, kF16>::go(a...) : F<4, kBF16>::go(a...);
}

// The division of a launch; false if the grid would be too large.
bool divide(const PagesStore &st, const PagesBatch &b, Work *w, unsigned *ctas) {
    w->L = 4;
    while (w->L * 8 < st.D) w->L *= 2;
    w->R = 32 / w->L;
    w->steps = (2 * st.H + w->R - 1) / w->R;
    // Measured, a warp a token and a warp a step: 16 x 2048 tokens of 8 x 128 into 8-bit
    // pages 84 and 140 us; 7900 fp32 tokens of 4 x 64 into 4-bit pages 13.6 and 17.0 us;
    // 16 single tokens 14.8 and 8.9 us.
    w->log_parts = 0;
    while ((1 << w->log_parts) < w->steps && ((int64_t)b.total << w->log_parts) < kSms * 16) ++w->log_parts;
    const int64_t n = (((int64_t)b.total << w->log_parts) + 7) / 8;
    *ctas = (unsigned)n;
    return n <= 0x7fffffff;
}

template <int BITS, int T> struct Write {
    static cudaError_t go(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
        Work w;
        unsigned ctas;
        if (!divide(st, b, &w, &ctas)) return cudaErrorInvalidValue;
        return launch_pdl(pages_write_kernel<BITS, T>, dim3(ctas), dim3(256), 0, s, true, st, b, x, w);
    }
};
template <int BITS, int T> struct Read {
    static cudaError_t go(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
        Work w;
        unsigned ctas;
        if (!divide(st, b, &w, &ctas)) return cudaErrorInvalidValue;
        return launch_pdl(pages_read_kernel<BITS, T>, dim3(ctas), dim3(256), 0, s, true, st, b, x, w);
    }
};

} // namespace

cudaError_t launch_pages_write(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
    if (b.total == 0 || b.batch == 0) return cudaSuccess;
    ProfScope prof("pages_write", s);
    count_launch();
    return by_type<Write>(st.bits, x.dtype, st, b, x, s);
}

cudaError_t launch_pages_read(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
    if (b.total == 0 || b.batch == 0) return cudaSuccess;
    ProfScope prof("pages_read", s);
    count_launch();
    return by_type<Read>(st.bits, x.dtype, st, b, x, s);
}

} // namespace kivi

// kivi_pages.cu -- writing new tokens into the paged store and reading them back.
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

// Eight consecutive elements at p, as floats.
template <class E> __device__ __forceinline__ void load8(const E *p, bool vec, float (&x)[8]) {
    if (vec) {
        constexpr int W = sizeof(E) / 2; // 16-byte words
        uint4 w[W];
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
        const E *e = reinterpret_cast<const E *>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f(p[i]);
    }
}
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

// One row of D elements belongs to L = D / 8 rounded up to a power of two lanes,
// eight elements each; a warp takes 32 / L of a token's 2 H rows (keys' heads,
// then values').
template <int BITS, int T>
__global__ void __launch_bounds__(256) pages_write_kernel(PagesStore st, PagesBatch b, PagesDense x, int L,
                                                          int wpt) {
    using E = typename Elem<T>::type;
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int tok = (int)(w / wpt);
    if (tok >= b.total) return;
    const int r = (int)(w % wpt) * (32 / L) + lane / L; // row of the token
    const int c = lane % L * 8;
    const bool live = r < 2 * st.H && c < st.D;
    const bool value = r >= st.H;
    const int head = value ? r - st.H : r;
    float e[8];
    const float inf = INFINITY;
    if (live)
        load8(static_cast<const E *>(value ? x.v : x.k) + tok * x.token + head * x.head + c, x.vec, e);
    const int i = find_sequence(b, tok);
    const Span s = pages_span(b, st, i);
    const int at = tok - s.start;
    const int t = s.kv - s.n + at;
    if (at < 0 || at >= s.n || t < 0) return; // warp-uniform
    const int page = pages_page(b, st, i, t);
    if (page < 0) return;
    const int64_t row = pages_row(st, page, head, t);
    unsigned char *dst = (value ? st.v : st.k) + row * st.row_bytes;
    if constexpr (BITS == 16) {
        if (!live) return;
        if (st.dtype == kBF16)
            store8(reinterpret_cast<__nv_bfloat16 *>(dst) + c, true, e);
        else
            store8(reinterpret_cast<__half *>(dst) + c, true, e);
    } else {
        constexpr float levels = (float)((1 << BITS) - 1);
        float mn = inf, mx = -inf;
        if (live) {
            mn = mx = e[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) {
                mn = fminf(mn, e[j]);
                mx = fmaxf(mx, e[j]);
            }
        }
        // lanes of another row never mix in: the butterfly stays within L lanes
        for (int o = L / 2; o > 0; o >>= 1) {
            const float a = __shfl_xor_sync(0xffffffffu, mn, o), z = __shfl_xor_sync(0xffffffffu, mx, o);
            mn = fminf(mn, a);
            mx = fmaxf(mx, z);
        }
        if (!live) return;
        const float span = __fsub_rn(mx, mn);
        const float scale = span == 0.0f ? 0.0f : __fdiv_rn(span, levels);
        uint32_t code[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float q = scale == 0.0f ? 0.0f : rintf(__fdiv_rn(__fsub_rn(e[j], mn), scale));
            q = fminf(fmaxf(q, 0.0f), levels);
            code[j] = __float_as_uint(__fadd_rn(q, 8388608.0f)) & 0xFFu;
        }
        if constexpr (BITS == 8) {
            uint2 o;
            o.x = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
            o.y = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
            *reinterpret_cast<uint2 *>(dst + c) = o;
        } else {
            uint32_t o = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) o |= code[j] << (4 * j);
            *reinterpret_cast<uint32_t *>(dst + c / 2) = o;
        }
        if (c == 0) (value ? st.vp : st.kp)[row] = make_float2(scale, mn);
    }
}

template <int BITS, int T>
__global__ void __launch_bounds__(256) pages_read_kernel(PagesStore st, PagesBatch b, PagesDense x, int L,
                                                         int wpt) {
    using E = typename Elem<T>::type;
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int tok = (int)(w / wpt);
    if (tok >= b.total) return;
    const int r = (int)(w % wpt) * (32 / L) + lane / L;
    const int c = lane % L * 8;
    const int i = find_sequence(b, tok);
    const Span s = pages_span(b, st, i);
    const int at = tok - s.start;
    const int t = s.kv - s.n + at;
    if (r >= 2 * st.H || c >= st.D || at < 0 || at >= s.n) return;
    const bool value = r >= st.H;
    const int head = value ? r - st.H : r;
    const int page = t < 0 ? -1 : pages_page(b, st, i, t);
    float e[8] = {};
    if (page >= 0) {
        const int64_t row = pages_row(st, page, head, t);
        const unsigned char *src = (value ? st.v : st.k) + row * st.row_bytes;
        if constexpr (BITS == 16) {
            if (st.dtype == kBF16)
                load8(reinterpret_cast<const __nv_bfloat16 *>(src) + c, true, e);
            else
                load8(reinterpret_cast<const __half *>(src) + c, true, e);
        } else {
            const float2 p = (value ? st.vp : st.kp)[row];
            if constexpr (BITS == 8) {
                const uint2 o = *reinterpret_cast<const uint2 *>(src + c);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    e[j] = fmaf((float)(((j < 4 ? o.x : o.y) >> (8 * (j & 3))) & 0xFFu), p.x, p.y);
            } else {
                const uint32_t o = *reinterpret_cast<const uint32_t *>(src + c / 2);
#pragma unroll
                for (int j = 0; j < 8; ++j) e[j] = fmaf((float)((o >> (4 * j)) & 15u), p.x, p.y);
            }
        }
    }
    E *dst = static_cast<E *>(const_cast<void *>(value ? x.v : x.k)) + tok * x.token + head * x.head + c;
    store8(dst, x.vec, e);
}

template <template <int, int> class F, class... A>
cudaError_t by_type(int bits, int dtype, A &&...a) {
    if (bits == 16)
        return dtype == kF32 ? F<16, kF32>::go(a...) : dtype == kF16 ? F<16, kF16>::go(a...) : F<16, kBF16>::go(a...);
    if (bits == 8)
        return dtype == kF32 ? F<8, kF32>::go(a...) : dtype == kF16 ? F<8, kF16>::go(a...) : F<8, kBF16>::go(a...);
    return dtype == kF32 ? F<4, kF32>::go(a...) : dtype == kF16 ? F<4, kF16>::go(a...) : F<4, kBF16>::go(a...);
}

// lanes per row and warps per token
struct RowSplit {
    int L, wpt;
    int64_t ctas;
    RowSplit(const PagesStore &st, const PagesBatch &b) {
        L = 4;
        while (L * 8 < st.D) L *= 2;
        wpt = (2 * st.H + 32 / L - 1) / (32 / L);
        ctas = ((int64_t)b.total * wpt + 7) / 8;
    }
};

template <int BITS, int T> struct Write {
    static cudaError_t go(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
        const RowSplit r(st, b);
        if (r.ctas > 0x7fffffff) return cudaErrorInvalidValue;
        return launch_pdl(pages_write_kernel<BITS, T>, dim3((unsigned)r.ctas), dim3(256), 0, s, false, st, b, x,
                          r.L, r.wpt);
    }
};
template <int BITS, int T> struct Read {
    static cudaError_t go(const PagesStore &st, const PagesBatch &b, const PagesDense &x, cudaStream_t s) {
        const RowSplit r(st, b);
        if (r.ctas > 0x7fffffff) return cudaErrorInvalidValue;
        return launch_pdl(pages_read_kernel<BITS, T>, dim3((unsigned)r.ctas), dim3(256), 0, s, false, st, b, x,
                          r.L, r.wpt);
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

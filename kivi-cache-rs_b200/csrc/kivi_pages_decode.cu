// kivi_pages_decode.cu -- one new token per sequence against its pages: the
// bandwidth-bound form of the paged attention, at most eight query heads per kv
// head.
//
// Per kv head and 16 tokens a warp forms S^T = K Q^T (m16n8k16: tokens x query
// heads) and O^T += V^T P^T (channels x query heads), so the eight columns are
// the query heads and nothing is padded to 16 rows.  Sums over channels (S) and
// over tokens (O) may run in any order, and so may O's rows: each lane takes the
// channels of K and V that let it read whole aligned vectors of a row straight
// into operand registers, and Q and the output follow the same order.  Nothing
// passes through shared memory; P^T comes out of S^T's accumulators by an 8 x 8
// transpose between lanes (movmatrix).
//
// Codes enter the products as the exact small integers c - 2^(b-1); a token's
// (scale s, zero z) apply to the sums, with z' = z + 2^(b-1) s:
//   q.k = s_k (q.c) + z'_k sum q,   o = sum (p s_v) c + sum p z'_v.
// P (or p s_v) is split into two 16-bit parts, so no weight is rounded to 8 or
// 11 bits: the tensor pipe has the room.  With codes the operands are f16, whose ten
// bits hold a code as it lies in its word (bf16's seven do not: twice the
// instructions); a row's query is scaled by a power of two into f16's upper end, and
// the weights by one that follows the tile's largest value scale up and, where O allows it,
// down, both undone in fp32.
//
// What bounds it: HBM for 16-bit pages (per token and kv head 4 D bytes, each read
// once: 16 x 32768 tokens of 8 x 128 in 318 us, 6.7 TB/s; under a window of 4096 and 4
// first tokens, 270 MB, 52 us).  For codes (2 D + 16 and D + 16 bytes) the work of taking
// them apart: 433 warp instructions per 16 tokens at 4 bits, 223 of them on the half-rate
// integer pipe, so 142 us for 396 MB (2.8 TB/s; issue slots 53% and that pipe 55% busy).
// More CTAs per SM (spills, or 16-token tiles) and larger tiles were no faster.
//
// Split: the visible tokens of all (sequence, kv head) rows form one flat list
// of tiles, and CTA i takes tiles [i per, (i + 1) per): one wave, no tail, any
// mix of lengths.  A row that spans CTAs leaves partial states (m, l, o) in the
// device's scratch (or the handle's workspace), and the CTA that finishes last joins them
// in CTA order, so
// the result does not depend on which one that is.
#include <math.h>

#include <algorithm>

#include "kivi_internal.cuh"
#include "kivi_pages.cuh"

namespace kivi {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxG = 8;
constexpr float kLazy = 8.0f; // a reference moves when a logit exceeds it by 2^8
constexpr int kKeep = 8;      // how far the value scales may fall before O's exponent follows

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// W bytes (2, 4, 8 or 16) at p into words w[0 .. (W + 3) / 4 - 1]; read once, so
// not kept in L1.
template <int W> __device__ __forceinline__ void load_words(const unsigned char *p, uint32_t *w) {
    if constexpr (W == 16)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "l"(p));
    else if constexpr (W == 8)
        asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else if constexpr (W == 4)
        asm volatile("ld.global.nc.L1::no_allocate.u32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    else {
        uint16_t h;
        asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(h) : "l"(p));
        w[0] = h;
    }
}
__device__ __forceinline__ float2 load_param(const float2 *p) {
    float2 r;
    asm volatile("ld.global.nc.v2.f32 {%0,%1}, [%2];" : "=f"(r.x), "=f"(r.y) : "l"(p));
    return r;
}

// A row's BYTES bytes, interleaved over LANES lanes in units of W bytes.
template <int LANES, int BYTES, int W>
__device__ __forceinline__ void load_row(const unsigned char *row, int lane, uint32_t *w) {
#pragma unroll
    for (int u = 0; u < BYTES / (LANES * W); ++u)
        load_words<W>(row + (u * LANES + lane) * W, w + u * ((W + 3) / 4));
}

template <bool F16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// (a, b) rounded to a 16-bit pair (a in the low half) and what the rounding left
template <bool F16> __device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    if constexpr (F16) {
        const __half2 h = __floats2half2_rn(a, b);
        const float2 f = __half22float2(h);
        const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
        hi = *reinterpret_cast<const uint32_t *>(&h);
        lo = *reinterpret_cast<const uint32_t *>(&r);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        hi = *reinterpret_cast<const uint32_t *>(&h);
        const __nv_bfloat162 r =
            __floats2bfloat162_rn(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
        lo = *reinterpret_cast<const uint32_t *>(&r);
    }
}

__device__ __forceinline__ uint32_t sub_h2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// Codes in the low bits of w's two halves (other bits ignored) as a pair of f16
// c - 2^(BITS-1), exact: the code in the mantissa of 1024.
template <int BITS> __device__ __forceinline__ uint32_t low_pair(uint32_t w) {
    if constexpr (BITS == 8) return sub_h2((w & 0x00ff00ffu) | 0x64006400u, 0x64806480u);
    return sub_h2((w & 0x000f000fu) | 0x64006400u, 0x64086408u);
}
// The next codes of the two halves.  8 bits: shifted down.  4 bits: left in place, so
// 16 (c - 8), the 16 taken out of the queries or of the output.
template <int BITS> __device__ __forceinline__ uint32_t next_pair(uint32_t w) {
    if constexpr (BITS == 8) return low_pair<8>(w >> 8);
    return sub_h2((w & 0x00f000f0u) | 0x64006400u, 0x64806480u);
}
// x in its upper end of f16: e with |x| 2^-e < 2^14 (-126 at least)
__device__ __forceinline__ int f16_exponent(uint32_t magnitude_bits) { return max(-126, (int)(magnitude_bits >> 23) - 140); }
__device__ __forceinline__ float exp2i(int k) { return __uint_as_float((uint32_t)(max(-126, min(127, k)) + 127) << 23); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Resident CTAs per SM: what the registers allow with no spill, or a small one (8 bits at
// head_dim 128: 108 bytes stored and 192 loaded; 4 bits at 96: 8 each).
__host__ __device__ constexpr int ctas_per_sm(int bits, int nd) { return nd == 4 || (bits < 16 && nd == 3) ? 3 : 4; }

// Geometry of the lanes' shares for head_dim D = 32 ND.
template <int BITS, int ND> struct Lay {
    static constexpr int D = 32 * ND;
    static constexpr int ROW = D * BITS / 8;
    static constexpr int largest(int n) { return n % 16 == 0 ? 16 : n % 8 == 0 ? 8 : n % 4 == 0 ? 4 : 2; }
    static constexpr int KB = ROW / 4, KU = largest(KB); // key bytes per lane and row, unit
    static constexpr int VB = ROW / 8, VU = largest(VB);
    static constexpr int KW = KB / 4;                                 // key words per row
    static constexpr int VW = VB / VU * ((VU + 3) / 4);               // value words per row
    static constexpr int TT = BITS == 16 ? 1 : 2;                     // 16-token subtiles per tile
    static constexpr int TK = 16 * TT;
    // channel of byte-offset `off` (within the lane's share) of lane `i` of n
    static constexpr __host__ __device__ int byte_at(int unit, int lanes, int i, int off) {
        return (off / unit * lanes + i) * unit + off % unit;
    }
    // channel that step s of S's sum (16 channels a step) has in register r, half e
    static __device__ __forceinline__ int kch(int s, int r, int e, int j) {
        if constexpr (BITS == 16) return byte_at(KU, 4, j, 8 * s + 4 * r) / 2 + e;
        if constexpr (BITS == 8) return byte_at(KU, 4, j, 4 * s) + 2 * e + r;
        return byte_at(KU, 4, j, 4 * (s >> 1)) * 2 + 2 * (s & 1) + r + 4 * e;
    }
    // channel of row g (half 0) or g + 8 (half 1) of O's m-tile mt
    static __device__ __forceinline__ int vch(int mt, int half, int g) {
        if constexpr (BITS == 16) return byte_at(VU, 8, g, 4 * mt) / 2 + half;
        if constexpr (BITS == 8) return byte_at(VU, 8, g, 2 * mt) + half;
        return byte_at(VU, 8, g, mt) * 2 + half;
    }
};

template <int BITS, int ND, bool F16> struct Tile {
    using L = Lay<BITS, ND>;
    uint32_t k[L::TT][2][L::KW];
    uint32_t v[L::TT][4][L::VW];
    float2 kp[L::TT][2], vp[L::TT][2]; // (scale, zero) of tokens g, g + 8
};

// A sequence's visible tiles: `ns` first ones, then tiles ws .. we - 1.
struct Tiles {
    int kv, lo, ns, ws, n;
};
template <int TK> __device__ __forceinline__ Tiles visible_tiles(const PagesAttn &a, const Span &s) {
    Tiles t;
    t.kv = s.n > 0 ? s.kv : 0;
    t.lo = a.window ? max(0, t.kv - a.window) : 0;
    t.ws = t.lo / TK;
    t.ns = min((min(a.sinks, t.lo) + TK - 1) / TK, t.ws);
    t.n = t.ns + (t.kv + TK - 1) / TK - t.ws;
    return t;
}

__device__ __forceinline__ void store_out(const PagesAttn &a, int tok, int hq, int c, float4 y, float l, float m) {
    y.x /= l, y.y /= l, y.z /= l, y.w /= l;
    uint2 w;
    if (a.dtype == kBF16) {
        const __nv_bfloat162 u = __floats2bfloat162_rn(y.x, y.y), v = __floats2bfloat162_rn(y.z, y.w);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&u), *reinterpret_cast<const uint32_t *>(&v));
    } else {
        const __half2 u = __floats2half2_rn(y.x, y.y), v = __floats2half2_rn(y.z, y.w);
        w = make_uint2(*reinterpret_cast<const uint32_t *>(&u), *reinterpret_cast<const uint32_t *>(&v));
    }
    uint16_t *d = static_cast<uint16_t *>(a.out) + tok * a.o_token + hq * a.o_head + c;
    if (a.o_vec) {
        *reinterpret_cast<uint2 *>(d) = w;
    } else {
        d[0] = (uint16_t)w.x, d[1] = (uint16_t)(w.x >> 16), d[2] = (uint16_t)w.y, d[3] = (uint16_t)(w.y >> 16);
    }
    if (a.lse && c == 0) a.lse[(int64_t)tok * a.Hq + hq] = m * 0.6931471805599453f + logf(l);
}

template <int BITS, int ND, bool F16>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(BITS, ND))
    pages_decode_kernel(const PagesAttn a, int min_per, int *counters) {
    static_assert(BITS == 16 || F16, "codes become f16 operands");
    using L = Lay<BITS, ND>;
    constexpr int D = L::D, TT = L::TT, TK = L::TK, STEPS = 2 * ND;
    // f16 weights over 16-bit pages are formed times 2^kBoost (below 2^15 with kLazy): what
    // f16's least step leaves of a small one is 2^-32 of the row's largest
    constexpr int kBoost = BITS == 16 && F16 ? 7 : 0;
    __shared__ long long s_sum[kWarps + 1];
    __shared__ long long s_base;
    __shared__ int s_seq, s_last;
    __shared__ float s_m[kWarps][kMaxG], s_l[kWarps][kMaxG];
    __shared__ float4 s_o4[kWarps][kMaxG][D / 4];
    __shared__ float s_w[kMaxG][64];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, j = lane & 3;
    const PagesStore &st = a.st;
    const int H = st.H, G = a.G;
    pdl_wait();
    pdl_trigger();

    // ---- the flat list: all tiles, this CTA's share, the sequence it starts in
    long long total = 0;
    for (int b0 = 0; b0 < a.b.batch; b0 += kThreads) {
        const int b = b0 + tid;
        if (b < a.b.batch) {
            const Span s = pages_span(a.b, st, b);
            const Tiles t = visible_tiles<TK>(a, s);
            total += t.n;
            if (t.n == 0 && s.n > 0 && b % gridDim.x == blockIdx.x) { // a row that sees nothing
                for (int r = 0; r < a.Hq; ++r) {
                    for (int c = 0; c < D; ++c)
                        static_cast<uint16_t *>(a.out)[s.start * a.o_token + r * a.o_head + c] = 0;
                    if (a.lse) a.lse[(int64_t)s.start * a.Hq + r] = -INFINITY;
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) s_sum[warp] = total;
    __syncthreads();
    total = 0;
    for (int w = 0; w < kWarps; ++w) total += s_sum[w];
    total *= H;
    long long per = (total + gridDim.x - 1) / gridDim.x;
    per = max(per, (long long)min_per);
    const long long begin = per * blockIdx.x, end = min(total, begin + per);
    if (begin >= end) return;
    long long run = 0; // tiles of earlier sequences, all heads
    for (int b0 = 0; b0 < a.b.batch; b0 += kThreads) {
        const int b = b0 + tid;
        const long long n = b < a.b.batch ? (long long)visible_tiles<TK>(a, pages_span(a.b, st, b)).n * H : 0;
        long long inc = n; // inclusive scan over the CTA
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        __syncthreads();
        if (lane == 31) s_sum[warp] = inc;
        __syncthreads();
        long long before = run;
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_sum[w];
            run += s_sum[w];
        }
        const long long first = before + inc - n;
        if (n > 0 && begin >= first && begin < first + n) {
            s_seq = b;
            s_base = first;
        }
        if (run > begin) break; // uniform: run is the same in every thread
    }
    __syncthreads();
    int b = s_seq;
    long long base = s_base;

    const float c2 = a.scale * 1.4426950408889634f;
    for (long long f = begin; f < end; ++b) {
        const Span sp = pages_span(a.b, st, b);
        const Tiles tl = visible_tiles<TK>(a, sp);
        const long long seq_tiles = (long long)tl.n * H;
        for (; f < end && f < base + seq_tiles;) {
            const int h = (int)((f - base) / tl.n);
            const long long row0 = base + (long long)h * tl.n;
            const int t0 = (int)(f - row0), t1 = (int)min((long long)tl.n, end - row0);
            f = row0 + t1;

            // ---- this row's queries, in the order of the key registers
            uint32_t qf[STEPS][2];
            float qs0 = 0.0f, qs1 = 0.0f; // sums of rows 2j, 2j + 1
            float c20 = c2, c21 = c2;     // their scores' exp2 units
            {
                const uint16_t *q = static_cast<const uint16_t *>(a.q) + sp.start * a.q_token +
                                    (int64_t)(h * G + g) * a.q_head;
                float sum = 0.0f;
#pragma unroll
                for (int s = 0; s < STEPS; ++s)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t x = 0;
                        if (g < G) x = q[L::kch(s, r, 0, j)] | (uint32_t)q[L::kch(s, r, 1, j)] << 16;
                        if (a.qsign < 0.0f) x ^= 0x80008000u;
                        qf[s][r] = x;
                    }
                if constexpr (BITS < 16) {
                    auto pair = [&](uint32_t x) {
                        if (a.dtype == kF16) return __half22float2(*reinterpret_cast<const __half2 *>(&x));
                        return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
                    };
                    float most = 0.0f;
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float2 y = pair(qf[s][r]);
                            most = fmaxf(most, fmaxf(fabsf(y.x), fabsf(y.y)));
                            sum += y.x + y.y;
                        }
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    const int e = f16_exponent(__float_as_uint(most));
                    const float f = exp2i(-e);
#pragma unroll
                    for (int s = 0; s < STEPS; ++s)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float2 y = pair(qf[s][r]);
                            const float fr = BITS == 4 && r ? f * 0.0625f : f; // next_pair's 16
                            const __half2 h = __floats2half2_rn(y.x * fr, y.y * fr);
                            qf[s][r] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                    c20 = c2 * exp2i(__shfl_sync(0xffffffffu, e, 8 * j));
                    c21 = c2 * exp2i(__shfl_sync(0xffffffffu, e, 8 * j + 4));
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    qs0 = __shfl_sync(0xffffffffu, sum, 8 * j);
                    qs1 = __shfl_sync(0xffffffffu, sum, 8 * j + 4);
                }
            }

            float o[STEPS][4];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
            float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f, z0 = 0.0f, z1 = 0.0f;
            int eref = -200; // exponent of O, with codes
            Tile<BITS, ND, F16> x;

            auto first_token = [&](int t) { return (t < tl.ns ? t : t - tl.ns + tl.ws) * TK; };
            auto pages_of = [&](int t, int (&pg)[TT]) {
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    const int tok = first_token(t) + 16 * s;
                    // a subtile that nobody sees may lie outside the table, or in a freed page
                    const bool any = tok < tl.kv && (tok + 16 > tl.lo || tok < a.sinks);
                    pg[s] = any ? max(pages_page(a.b, st, b, tok), 0) : 0;
                }
            };
            auto load_k = [&](int t, const int (&pg)[TT]) {
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    const int64_t r = pages_row(st, pg[s], h, first_token(t) + 16 * s);
                    const unsigned char *p = st.k + (r + g) * L::ROW;
                    load_row<4, L::ROW, L::KU>(p, j, x.k[s][0]);
                    load_row<4, L::ROW, L::KU>(p + 8 * L::ROW, j, x.k[s][1]);
                    if constexpr (BITS < 16) {
                        x.kp[s][0] = load_param(st.kp + r + g);
                        x.kp[s][1] = load_param(st.kp + r + g + 8);
                    }
                }
            };
            auto load_v = [&](int t, const int (&pg)[TT]) {
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    const int64_t r = pages_row(st, pg[s], h, first_token(t) + 16 * s);
                    const unsigned char *p = st.v + (r + 2 * j) * L::ROW;
                    load_row<8, L::ROW, L::VU>(p, g, x.v[s][0]);
                    load_row<8, L::ROW, L::VU>(p + L::ROW, g, x.v[s][1]);
                    load_row<8, L::ROW, L::VU>(p + 8 * L::ROW, g, x.v[s][2]);
                    load_row<8, L::ROW, L::VU>(p + 9 * L::ROW, g, x.v[s][3]);
                    if constexpr (BITS < 16) {
                        x.vp[s][0] = load_param(st.vp + r + g);
                        x.vp[s][1] = load_param(st.vp + r + g + 8);
                    }
                }
            };

            int t = t0 + warp;
            int pg[TT], pn[TT];
            if (t < t1) {
                pages_of(t, pg);
                load_k(t, pg);
                load_v(t, pg);
                if (t + kWarps < t1) pages_of(t + kWarps, pn);
            }
            for (; t < t1; t += kWarps) {
                const bool more = t + kWarps < t1;
                const int tok = first_token(t);
                const bool edge = tok + TK > tl.kv || (tok < tl.lo && tok + TK > a.sinks);
                auto seen = [&](int u) { return u < tl.kv && (u >= tl.lo || u < a.sinks); };
                // ---- S^T and the logits in exp2 units: tokens g, g + 8 x rows 2j, 2j + 1
                float sx[TT][4];
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        uint32_t a0, a1, a2, a3;
                        if constexpr (BITS == 16) {
                            a0 = x.k[s][0][2 * i], a2 = x.k[s][0][2 * i + 1];
                            a1 = x.k[s][1][2 * i], a3 = x.k[s][1][2 * i + 1];
                        } else if constexpr (BITS == 8) {
                            a0 = low_pair<8>(x.k[s][0][i]), a2 = next_pair<8>(x.k[s][0][i]);
                            a1 = low_pair<8>(x.k[s][1][i]), a3 = next_pair<8>(x.k[s][1][i]);
                        } else {
                            const uint32_t u = x.k[s][0][i / 2] >> (8 * (i & 1)), w = x.k[s][1][i / 2] >> (8 * (i & 1));
                            a0 = low_pair<4>(u), a2 = next_pair<4>(u);
                            a1 = low_pair<4>(w), a3 = next_pair<4>(w);
                        }
                        mma<F16>(c, a0, a1, a2, a3, qf[i][0], qf[i][1]);
                    }
                    if constexpr (BITS == 16) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sx[s][i] = c[i] * c2;
                    } else {
                        constexpr float half = (float)(1 << (BITS - 1));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float z = fmaf(half, x.kp[s][i].x, x.kp[s][i].y) * c2;
                            sx[s][2 * i] = fmaf(x.kp[s][i].x * c20, c[2 * i], z * qs0);
                            sx[s][2 * i + 1] = fmaf(x.kp[s][i].x * c21, c[2 * i + 1], z * qs1);
                        }
                    }
                }
                float2 vp[TT][2];
                if constexpr (BITS < 16) {
#pragma unroll
                    for (int s = 0; s < TT; ++s) vp[s][0] = x.vp[s][0], vp[s][1] = x.vp[s][1];
                }
                if (edge) {
#pragma unroll
                    for (int s = 0; s < TT; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (!seen(tok + 16 * s + g + 8 * i)) {
                                sx[s][2 * i] = sx[s][2 * i + 1] = -INFINITY;
                                vp[s][i] = make_float2(0.0f, 0.0f);
                            }
                }
                if (more) load_k(t + kWarps, pn);
                // ---- the running reference
                float t0x = sx[0][0], t1x = sx[0][1];
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    t0x = fmaxf(t0x, fmaxf(sx[s][0], sx[s][2]));
                    t1x = fmaxf(t1x, fmaxf(sx[s][1], sx[s][3]));
                }
                if (__any_sync(0xffffffffu, t0x > m0 + kLazy || t1x > m1 + kLazy)) {
#pragma unroll
                    for (int k = 4; k < 32; k <<= 1) {
                        t0x = fmaxf(t0x, __shfl_xor_sync(0xffffffffu, t0x, k));
                        t1x = fmaxf(t1x, __shfl_xor_sync(0xffffffffu, t1x, k));
                    }
                    const float n0 = fmaxf(m0, t0x), n1 = fmaxf(m1, t1x);
                    const float f0 = n0 == -INFINITY ? 1.0f : ex2(m0 - n0), f1 = n1 == -INFINITY ? 1.0f : ex2(m1 - n1);
                    m0 = n0, m1 = n1;
                    l0 *= f0, z0 *= f0, l1 *= f1, z1 *= f1;
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) o[i][0] *= f0, o[i][2] *= f0, o[i][1] *= f1, o[i][3] *= f1;
                }
                float fv = 1.0f; // of the value scales
                if constexpr (BITS < 16) {
                    uint32_t most = 0;
#pragma unroll
                    for (int s = 0; s < TT; ++s)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t b = __float_as_uint(fabsf(vp[s][i].x));
                            if (b < 0x7f800000u) most = max(most, b);
                        }
                    most = __reduce_max_sync(0xffffffffu, most);
                    // p <= 2^kLazy: weights below 2^14.  O follows the scales both ways (down
                    // as far as fp32 lets it), so that large ones of small weight take nothing
                    // from later tiles.
                    const int e = f16_exponent(most) + (int)kLazy;
                    if (e > eref || (e + kKeep < eref && most > 0)) {
                        int n = e;
                        if (e < eref) {
                            uint32_t big = 0;
#pragma unroll
                            for (int i = 0; i < STEPS; ++i)
#pragma unroll
                                for (int k = 0; k < 4; ++k) big = max(big, __float_as_uint(fabsf(o[i][k])));
                            big = __reduce_max_sync(0xffffffffu, big);
                            if (big > 0 && big < 0x7f800000u) n = min(max(e, eref + (int)(big >> 23) - 227), eref); // below 2^101
                        }
                        const int d = eref - n, h = d >> 1;
                        const float f0 = exp2i(h), f1 = exp2i(d - h);
                        eref = n;
#pragma unroll
                        for (int i = 0; i < STEPS; ++i)
#pragma unroll
                            for (int k = 0; k < 4; ++k) o[i][k] = o[i][k] * f0 * f1;
                    }
                    fv = exp2i(-eref);
                }
                const float r0 = (m0 == -INFINITY ? 0.0f : m0) - kBoost, r1 = (m1 == -INFINITY ? 0.0f : m1) - kBoost;
                // ---- weights, and O^T += V^T P^T
#pragma unroll
                for (int s = 0; s < TT; ++s) {
                    float p[4] = {ex2(sx[s][0] - r0), ex2(sx[s][1] - r1), ex2(sx[s][2] - r0), ex2(sx[s][3] - r1)};
                    l0 += p[0] + p[2];
                    l1 += p[1] + p[3];
                    if constexpr (BITS < 16) {
                        constexpr float half = (float)(1 << (BITS - 1));
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float z = fmaf(half, vp[s][i].x, vp[s][i].y);
                            z0 = fmaf(p[2 * i], z, z0);
                            z1 = fmaf(p[2 * i + 1], z, z1);
                            p[2 * i] *= vp[s][i].x * fv;
                            p[2 * i + 1] *= vp[s][i].x * fv;
                        }
                    }
                    uint32_t h0, e0, h1, e1;
                    split2<F16>(p[0], p[1], h0, e0);
                    split2<F16>(p[2], p[3], h1, e1);
                    h0 = transpose8(h0), h1 = transpose8(h1), e0 = transpose8(e0), e1 = transpose8(e1);
                    if (BITS == 16 && edge) { // 0 times what an unseen row holds is not 0 where that is not finite
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!seen(tok + 16 * s + 2 * j + (i & 1) + 8 * (i >> 1)))
#pragma unroll
                                for (int w = 0; w < L::VW; ++w) x.v[s][i][w] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        uint32_t a0, a1, a2, a3;
                        if constexpr (BITS == 16) {
                            a0 = prmt(x.v[s][0][i], x.v[s][1][i], 0x5410), a1 = prmt(x.v[s][0][i], x.v[s][1][i], 0x7632);
                            a2 = prmt(x.v[s][2][i], x.v[s][3][i], 0x5410), a3 = prmt(x.v[s][2][i], x.v[s][3][i], 0x7632);
                        } else if constexpr (BITS == 8) {
                            const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
                            const uint32_t u = prmt(x.v[s][0][i / 2], x.v[s][1][i / 2], sel);
                            const uint32_t w = prmt(x.v[s][2][i / 2], x.v[s][3][i / 2], sel);
                            a0 = low_pair<8>(u), a1 = next_pair<8>(u);
                            a2 = low_pair<8>(w), a3 = next_pair<8>(w);
                        } else {
                            constexpr bool two = L::VU > 2; // two half words of four channels per word
                            const int wi = two ? i / 4 : i / 2;
                            const uint32_t sel = two && (i & 2) ? 0x7632 : 0x5410;
                            const uint32_t u = prmt(x.v[s][0][wi], x.v[s][1][wi], sel) >> (8 * (i & 1));
                            const uint32_t w = prmt(x.v[s][2][wi], x.v[s][3][wi], sel) >> (8 * (i & 1));
                            a0 = low_pair<4>(u), a1 = next_pair<4>(u);
                            a2 = low_pair<4>(w), a3 = next_pair<4>(w);
                        }
                        mma<F16>(o[i], a0, a1, a2, a3, e0, e1);
                        mma<F16>(o[i], a0, a1, a2, a3, h0, h1);
                    }
                }
                if (more) {
                    load_v(t + kWarps, pn);
                    if (t + 2 * kWarps < t1) pages_of(t + 2 * kWarps, pn);
                }
            }

            // ---- join the warps
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, k);
                l1 += __shfl_xor_sync(0xffffffffu, l1, k);
                z0 += __shfl_xor_sync(0xffffffffu, z0, k);
                z1 += __shfl_xor_sync(0xffffffffu, z1, k);
            }
            __syncthreads(); // the last segment's reads
            if (g == 0) {
                s_m[warp][2 * j] = m0, s_m[warp][2 * j + 1] = m1;
                s_l[warp][2 * j] = l0 * exp2i(-kBoost), s_l[warp][2 * j + 1] = l1 * exp2i(-kBoost);
            }
            {
                const float fo[2] = {BITS < 16 ? exp2i(eref) : exp2i(-kBoost),
                                     BITS < 16 ? exp2i(eref) * (BITS == 4 ? 0.0625f : 1.0f) : exp2i(-kBoost)};
                float *r0p = reinterpret_cast<float *>(s_o4[warp][2 * j]), *r1p = reinterpret_cast<float *>(s_o4[warp][2 * j + 1]);
#pragma unroll
                for (int i = 0; i < STEPS; ++i)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int c = L::vch(i, e, g);
                        r0p[c] = fmaf(o[i][2 * e], fo[e], z0);
                        r1p[c] = fmaf(o[i][2 * e + 1], fo[e], z1);
                    }
            }
            __syncthreads();
            const int c0 = (int)(row0 / per), c1 = (int)((row0 + tl.n - 1) / per);
            const bool whole = c0 == c1;
            constexpr int PF4 = D / 4;
            constexpr int64_t kPart = kMaxG * (D + 2);
            const bool started = c0 == (int)blockIdx.x;
            float *part = a.part + ((int64_t)blockIdx.x * 2 + (started ? 1 : 0)) * kPart;
            for (int i = tid; i < G * PF4; i += kThreads) {
                const int r = i / PF4, c = i % PF4;
                float mm = s_m[0][r];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float l = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    // a warp without tiles left m at -inf
                    const float fw = s_m[w][r] == -INFINITY ? (mm == -INFINITY ? 1.0f : 0.0f) : ex2(s_m[w][r] - mm);
                    const float4 y = s_o4[w][r][c];
                    acc.x = fmaf(fw, y.x, acc.x), acc.y = fmaf(fw, y.y, acc.y);
                    acc.z = fmaf(fw, y.z, acc.z), acc.w = fmaf(fw, y.w, acc.w);
                    l = fmaf(fw, s_l[w][r], l);
                }
                if (whole) {
                    store_out(a, sp.start, h * G + r, 4 * c, acc, l, mm);
                } else {
                    reinterpret_cast<float4 *>(part)[i] = acc;
                    if (c == 0) {
                        part[kMaxG * D + 2 * r] = mm;
                        part[kMaxG * D + 2 * r + 1] = l;
                    }
                }
            }
            if (whole) continue;
            // ---- the last CTA of the row joins its parts, in CTA order
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicAdd(counters + c0, 1) == c1 - c0;
            __syncthreads();
            if (!s_last) continue;
            if (tid == 0) counters[c0] = 0; // for the next call
            __threadfence();
            const int parts = c1 - c0 + 1;
            const float *first = a.part;
            auto part_of = [&](int k) { return first + ((int64_t)(c0 + k) * 2 + (k == 0 ? 1 : 0)) * kPart; };
            for (int i0 = 0; i0 < G * PF4; i0 += kThreads) {
                const int i = i0 + tid;
                const bool live = i < G * PF4;
                const int r = live ? i / PF4 : 0;
                float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float mm = -INFINITY, l = 0.0f;
                for (int k0 = 0; k0 < parts; k0 += 64) {
                    const int kn = min(64, parts - k0);
                    __syncthreads();
                    for (int e = tid; e < G * kn; e += kThreads)
                        s_w[e / kn][e % kn] = __ldcg(part_of(k0 + e % kn) + kMaxG * D + 2 * (e / kn));
                    __syncthreads();
                    if (!live) continue;
                    float nm = mm;
                    for (int k = 0; k < kn; ++k) nm = fmaxf(nm, s_w[r][k]);
                    const float ref = nm == -INFINITY ? 0.0f : nm;
                    const float fo = ex2(mm - ref);
                    acc.x *= fo, acc.y *= fo, acc.z *= fo, acc.w *= fo, l *= fo;
                    mm = nm;
#pragma unroll 8
                    for (int k = 0; k < kn; ++k) {
                        const float fw = ex2(s_w[r][k] - ref);
                        const float *pk = part_of(k0 + k);
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(pk) + i);
                        l = fmaf(fw, __ldcg(pk + kMaxG * D + 2 * r + 1), l);
                        acc.x = fmaf(fw, y.x, acc.x), acc.y = fmaf(fw, y.y, acc.y);
                        acc.z = fmaf(fw, y.z, acc.z), acc.w = fmaf(fw, y.w, acc.w);
                    }
                }
                if (live) store_out(a, sp.start, h * G + r, 4 * (i % PF4), acc, l, mm);
            }
        }
        base += seq_tiles;
    }
}

template <int BITS, int ND, bool F16>
cudaError_t launch_decode(const PagesAttn &a, cudaStream_t s) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    const int grid = sms * ctas_per_sm(BITS, ND);
    int *counters = reinterpret_cast<int *>(a.part + a.part_floats) - kPagesCounters;
    if (grid > kPagesCounters || (int64_t)grid * 2 * kMaxG * (32 * ND + 2) > a.part_floats - kPagesCounters)
        return cudaErrorInvalidConfiguration;
    // a CTA takes at least two tiles per warp: fewer make more parts to join (one sequence
    // of 4096 8-bit tokens: 16.6 us with two, 16.1 us with one, 20.9 us with four)
    return launch_pdl(pages_decode_kernel<BITS, ND, F16>, dim3((unsigned)grid), dim3(kThreads), 0, s, true, a,
                      2 * kWarps, counters);
}

template <int BITS, bool F16> cudaError_t by_dim(const PagesAttn &a, cudaStream_t s) {
    switch (a.st.D) {
    case 32: return launch_decode<BITS, 1, F16>(a, s);
    case 64: return launch_decode<BITS, 2, F16>(a, s);
    case 96: return launch_decode<BITS, 3, F16>(a, s);
    default: return launch_decode<BITS, 4, F16>(a, s);
    }
}

} // namespace

int64_t pages_decode_scratch(int sms) { return (int64_t)sms * 4 * 2 * kMaxG * (128 + 2); }

bool pages_decode_supported(const PagesAttn &a) { return a.b.most == 1 && a.G <= kMaxG; }

cudaError_t launch_pages_decode(const PagesAttn &a, cudaStream_t s) {
    ProfScope prof("pages_decode", s);
    count_launch();
    const bool f16 = a.dtype == kF16;
    switch (a.st.bits) {
    case 16: return f16 ? by_dim<16, true>(a, s) : by_dim<16, false>(a, s);
    case 8: return by_dim<8, true>(a, s);
    default: return by_dim<4, true>(a, s);
    }
}

} // namespace kivi

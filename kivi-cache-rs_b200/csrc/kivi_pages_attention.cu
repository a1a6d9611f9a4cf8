// kivi_pages_attention.cu -- causal attention of a batch's newest tokens over
// the paged store.
#include <math.h>

#include <algorithm>

#include "kivi_internal.cuh"
#include "kivi_pages.cuh"

namespace kivi {
namespace {

__device__ __forceinline__ float elem(const void *p, int dtype, int64_t i) {
    return dtype == kBF16 ? __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i])
                          : __half2float(static_cast<const __half *>(p)[i]);
}

// Channel c of the row at `row` of one side of the store.
__device__ __forceinline__ float stored(const PagesStore &st, bool value, int64_t row, int c, float2 p) {
    const unsigned char *r = (value ? st.v : st.k) + row * st.row_bytes;
    if (st.bits == 16) return elem(r, st.dtype, c);
    const uint32_t code = st.bits == 8 ? r[c] : (r[c / 2] >> (4 * (c & 1))) & 15u;
    return fmaf((float)code, p.x, p.y);
}

// One warp per (query row, query head): lanes share the channels, one token at
// a time with a running maximum and sum.
__global__ void __launch_bounds__(128) pages_rows_kernel(PagesAttn a) {
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int hq = (int)(w % a.Hq);
    const int64_t r = w / a.Hq;
    const int i = (int)(r / a.b.most);
    if (i >= a.b.batch) return;
    const Span s = pages_span(a.b, a.st, i);
    const int at = (int)(r % a.b.most);
    if (at >= s.n) return;
    const int head = hq / a.G, D = a.st.D;
    const int p = s.kv - s.n + at;
    const int64_t tok = s.start + at;
    float q[4], o[4] = {}, m = -INFINITY, l = 0.0f;
    for (int j = 0; j < 4; ++j) {
        const int c = lane + 32 * j;
        q[j] = c < D ? elem(a.q, a.dtype, tok * a.q_token + hq * a.q_head + c) * a.qsign : 0.0f;
    }
    const float c2 = a.scale * 1.4426950408889634f;
    const int lo = a.window ? max(0, p - a.window + 1) : 0;
    int64_t base = 0;
    for (int t = min(a.sinks, lo) > 0 ? 0 : lo; t <= p; ++t) {
        if (t < lo && t >= a.sinks) t = lo;
        const int page = pages_page(a.b, a.st, i, t);
        base = pages_row(a.st, max(page, 0), head, t);
        const float2 kp = a.st.bits == 16 ? make_float2(0, 0) : a.st.kp[base];
        const float2 vp = a.st.bits == 16 ? make_float2(0, 0) : a.st.vp[base];
        float x = 0.0f;
        for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < D) x = fmaf(q[j], stored(a.st, false, base, lane + 32 * j, kp), x);
        for (int k = 16; k > 0; k >>= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
        x *= c2;
        const float nm = fmaxf(m, x);
        const float ref = nm == -INFINITY ? 0.0f : nm;
        const float f = exp2f(m - ref), e = exp2f(x - ref);
        m = nm;
        l = l * f + e;
        for (int j = 0; j < 4; ++j)
            if (lane + 32 * j < D) o[j] = fmaf(e, stored(a.st, true, base, lane + 32 * j, vp), o[j] * f);
    }
    for (int j = 0; j < 4; ++j) {
        const int c = lane + 32 * j;
        if (c >= D) continue;
        const float y = p < 0 ? 0.0f : o[j] / l;
        const int64_t d = tok * a.o_token + hq * a.o_head + c;
        if (a.dtype == kBF16)
            static_cast<__nv_bfloat16 *>(a.out)[d] = __float2bfloat16_rn(y);
        else
            static_cast<__half *>(a.out)[d] = __float2half_rn(y);
    }
    if (a.lse && lane == 0) a.lse[tok * a.Hq + hq] = p < 0 ? -INFINITY : m * 0.6931471805599453f + logf(l);
}

} // namespace

cudaError_t pages_scratch_floats(const PagesStore &st, int64_t *floats) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    *floats = std::max((int64_t)sms * 4 * 2 * 8 * (st.D + 2), pages_chunk_scratch(st.D, sms)) + kPagesCounters;
    return e;
}

cudaError_t launch_pages_attention(const PagesAttn &a, cudaStream_t s) {
    if (a.b.total == 0 || a.b.batch == 0 || a.b.most == 0) return cudaSuccess;
    if (pages_decode_supported(a)) return launch_pages_decode(a, s);
    if (pages_chunk_supported(a)) return launch_pages_chunk(a, s);
    const int64_t warps = (int64_t)a.b.batch * a.b.most * a.Hq;
    const int64_t ctas = (warps + 3) / 4;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    ProfScope prof("pages_attention", s);
    count_launch();
    return launch_pdl(pages_rows_kernel, dim3((unsigned)ctas), dim3(128), 0, s, false, a);
}

} // namespace kivi

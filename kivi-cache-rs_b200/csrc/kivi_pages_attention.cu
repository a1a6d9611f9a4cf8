// kivi_pages_attention.cu -- which kernel a paged attention call takes, and the
// scratch they share.
#include <algorithm>

#include "kivi_internal.cuh"
#include "kivi_pages.cuh"

namespace kivi {

cudaError_t pages_scratch_floats(int64_t *floats) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    *floats = std::max(pages_decode_scratch(sms), pages_chunk_scratch(sms)) + kPagesCounters;
    return e;
}

bool pages_attention_supported(const PagesAttn &a) { return pages_decode_supported(a) || pages_chunk_supported(a); }

// One newest token per sequence and at most eight query heads per kv head: the decode
// kernel, whose eight matrix columns those heads are.  Measured against the chunk
// kernel, most of whose 128 rows such a call leaves empty: 16 x 32768 bf16 tokens 316
// and 329 us; ragged 4-bit up to 65521 tokens, 8 heads a kv head, 140 and 597 us; one
// sequence of 4096 8-bit tokens 18.7 and 17.7 us.  Anything else: the chunk kernel.
cudaError_t launch_pages_attention(const PagesAttn &a, cudaStream_t s) {
    if (a.b.total == 0 || a.b.batch == 0 || a.b.most == 0) return cudaSuccess;
    return pages_decode_supported(a) ? launch_pages_decode(a, s) : launch_pages_chunk(a, s);
}

} // namespace kivi

// kivi_pages.cuh -- the paged key/value store: layout, batches and the kernel
// launchers shared by its translation units.
//
// A store of P pages holds, for keys and for values, rows of head_dim elements
//   data   [P][H][page][row_bytes]   row_bytes = D * bits / 8
//   params [P][H][page]              float2 (scale, zero), codes only
// 16-bit rows are the elements as they came; 8- and 4-bit rows are codes, first
// channel in the low bits (the per-token stream order of quant.rs:330-377 with
// one group per row), each standing for fma(code, scale, zero).  A (page, head)
// block is contiguous, so one copy brings any run of a page's tokens in, and
// neither order nor place of a sequence's pages matters.
//
// A batch names, per sequence, its pages (a block-table row), its tokens
// (kv_lens) and how many of them are the call's own newest ones (cu_tokens, the
// offsets of their rows in the dense arrays).  All three live in device memory,
// so a step needs no host synchronisation and can be captured.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace kivi {

enum DType { kF32 = 0, kF16 = 1, kBF16 = 2 };
inline int dtype_bytes(int t) { return t == kF32 ? 4 : 2; }

// What a kernel found wrong with the device-side batch (kivi_pages_status).
constexpr unsigned kPagesBadPage = 1u;    // a page number outside the store
constexpr unsigned kPagesBadLengths = 2u; // offsets or lengths outside their arrays
constexpr unsigned kPagesGaveUp = 4u;     // a bounded wait ran out

struct PagesStore {
    int bits;       // 16, 8, 4
    int dtype;      // element type of 16-bit rows (kF16, kBF16)
    int H, D;
    int page, shift; // tokens per page (a power of two) and its logarithm
    int num_pages;
    int row_bytes;
    unsigned char *k, *v;
    float2 *kp, *vp;
    unsigned int *status;
};

struct PagesBatch {
    const int32_t *table; // [batch][table_stride], `width` entries of a row used
    int64_t table_stride;
    int width;
    const int32_t *cu;      // [batch + 1]
    const int32_t *kv_lens; // [batch]
    int batch;
    int total; // rows of the dense arrays
    int most;  // most newest tokens of any sequence
};

// Dense rows [total][heads][D]: element strides of a token and of a head.
struct PagesDense {
    const void *k, *v;
    int64_t token, head;
    int dtype;
    bool vec; // rows start on 16-byte boundaries
};

// Tensor maps of 16-bit pages (host memory; passed to the kernel by value).
struct PagesMaps {
    CUtensorMap k, v;
};

struct PagesAttn {
    PagesStore st;
    PagesBatch b;
    const void *q;
    int64_t q_token, q_head; // element strides
    bool q_vec;
    void *out;
    int64_t o_token, o_head;
    bool o_vec;
    float *lse; // [total][Hq] or null
    int dtype;
    int Hq, G;          // query heads, query heads per kv head
    float scale;        // >= 0; a negative scale is folded into qsign
    float qsign;
    int window, sinks;  // window 0: everything up to the row's own token
    float *part;        // the device's scratch
    int64_t part_floats;
    const PagesMaps *maps;
};

// One sequence's span, clamped to its arrays: rows [start, start + n) of the
// dense arrays are its tokens kv - n .. kv - 1.
struct Span {
    int start, n, kv;
};
__device__ __forceinline__ Span pages_span(const PagesBatch &b, const PagesStore &st, int i) {
    const int s0 = __ldg(b.cu + i), s1 = __ldg(b.cu + i + 1), kv0 = __ldg(b.kv_lens + i);
    Span s;
    s.start = min(max(s0, 0), b.total);
    s.n = min(min(max(s1, s.start), b.total) - s.start, b.most);
    s.kv = (int)min((int64_t)max(kv0, 0), (int64_t)b.width << st.shift);
    if (s.start != s0 || s.start + s.n != s1 || s.kv != kv0) atomicOr(st.status, kPagesBadLengths);
    return s;
}

// Block index (page * H + head-less) of token t of sequence i: the page number,
// 0 where the table names none of the store's (reported).
__device__ __forceinline__ int pages_page(const PagesBatch &b, const PagesStore &st, int i, int t) {
    const int p = __ldg(b.table + (int64_t)i * b.table_stride + (t >> st.shift));
    if ((unsigned)p >= (unsigned)st.num_pages) {
        atomicOr(st.status, kPagesBadPage);
        return -1;
    }
    return p;
}

// Row index (into [P][H][page]) of a token's slot.
__device__ __forceinline__ int64_t pages_row(const PagesStore &st, int page, int head, int t) {
    return ((((int64_t)page * st.H + head) << st.shift)) + (t & (st.page - 1));
}

cudaError_t launch_pages_write(const PagesStore &st, const PagesBatch &b, const PagesDense &x,
                               cudaStream_t s);
cudaError_t launch_pages_read(const PagesStore &st, const PagesBatch &b, const PagesDense &x,
                              cudaStream_t s);
cudaError_t launch_pages_attention(const PagesAttn &a, cudaStream_t s);
// Scratch of launch_pages_attention on the current device, for any store: partial
// states, then kPagesCounters counters, zeroed once and left zero by every call.
constexpr int kPagesCounters = 2048;
cudaError_t pages_scratch_floats(int64_t *floats);
bool pages_attention_supported(const PagesAttn &a);
// One newest token per sequence, at most eight query heads per kv head
// (kivi_pages_decode.cu).
bool pages_decode_supported(const PagesAttn &a);
int64_t pages_decode_scratch(int sms); // floats
// Anything else (kivi_pages_chunk.cu).
bool pages_chunk_supported(const PagesAttn &a);
int64_t pages_chunk_scratch(int sms); // floats
cudaError_t pages_tensor_maps(const PagesStore &st, PagesMaps *maps);
cudaError_t launch_pages_chunk(const PagesAttn &a, cudaStream_t s);
cudaError_t launch_pages_decode(const PagesAttn &a, cudaStream_t s);

} // namespace kivi

// kivi_pages_chunk.cu -- several new tokens per sequence (prompt chunks, drafts)
// or many query heads per kv head against the paged store, on the
// 5th-generation tensor cores.
//
// A block is the packed query rows (token, head of the kv head's group) of up to
// 256 / G consecutive new tokens: two row tiles, A and B, of 128.  Per 128
// cached tokens
//   S = Q K^T  tcgen05.mma, M = N = 128, Q and K in shared memory (128-byte
//              swizzle, K-major), S in tensor memory;
//   softmax    one thread per row: its S row from tensor memory, running maximum
//              and sum in fp32, P (16 bits) back over S;
//   O += P V   P from tensor memory, V in shared memory as it lies in the page
//              ([token][channel] = MN-major), O in tensor memory.
// The tiles A and B take turns: while one's softmax runs, the tensor pipe does
// the other's O += P V and its next S.  A block of at most 128 rows has one row
// tile; A then takes its even and B its odd cached tiles, and their states are
// joined at the end (tensor memory lanes are the rows, so A's threads read B's O
// from their own lanes).
//
// The maximum that P refers to moves only when a row exceeds it by 2^8: P stays
// within its type and O is rarely rescaled.  A row sees tokens by its position;
// unseen scores are replaced by -inf and weigh 0, and in tiles of which some row does not
// see some token, V rows that nobody sees are zeroed and infinities and NaN are taken
// out before O += P V (0 times infinity is not 0) and added to the rows that do
// see them apart.
//
// Rounded below fp32: P, to the operand type, and codes' keys and values, to f16, once.
// P in two parts, as the decode kernel has it, would double O += P V, a half of the tensor
// pipe's work; error against 64 bits of a 2048-token chunk's bf16 outputs 0.0023, of which
// their own rounding is 0.0017.
//
// Work split: blocks x kv heads x cached tiles form one flat list, and each of
// the persistent CTAs (one per SM) takes an equal run of it: no last wave, any
// mix of lengths.  A (block, head) that spans CTAs leaves partial states in the
// device's scratch (or the handle's workspace); the CTA that finishes last joins them in
// CTA order.
//
// Warps: 0-3 softmax of A, 4-7 of B, 8 MMA issue, 9 the run's segments and the copies
// (TMA tensor maps over the pages, a box per page and 64 channels), 10-11 the masked
// tiles' V rows.  8- and 4-bit pages: instead of copies, warps 10-15 turn the codes into
// f16 operand tiles in shared memory, each tile's keys and values scaled by a power of
// two into f16's upper end (undone in the softmax's factor and O's exponent, which moves
// with the values').
//
// What bounds it: per cached tile and pair of row tiles the tensor pipe has 2048 cycles
// of work and the special function unit as many exponentials (three quarters of them
// stay there, one quarter are polynomials on the FMA pipe), but a row tile's chain S ->
// softmax -> P V -> next S is about 3400: a 2048-token chunk over 10240 bf16 tokens, 32
// heads over 8, takes 297 us in short bursts and 340 us back to back (1.04 and 0.91
// PFLOP/s, tensor pipe 49% active), an 8192-token prompt under a window of 1024 256 us: a
// block there is ten tiles, some 34000 cycles, and 5000 for queries in and 4500 for rows out
// beside them, three of the tiles masked.  With 8-bit pages ragged 1024-token
// chunks over 8000 take 725 us (0.53 PFLOP/s): the converting warps share the issue slots
// with the softmax (of 709 us, 529 were left without the conversion's arithmetic and 457
// without its loads as well).
// Measured and left out, when the chunk above took 291: 16 softmax warps, two to a row
// (301-319 us); S in halves of 64 tokens, double-buffered (310 us; 416 us with the next
// half's maximum taken between the exponentials); half or none of the exponentials on the
// FMA pipe (314 us each).
#include <cudaTypedefs.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kivi_internal.cuh"
#include "kivi_pages.cuh"

namespace kivi {
namespace {

constexpr int kTok = 128;                 // cached tokens per tile
constexpr int kRows = 128;                // rows of one row tile
constexpr int kSoft = 8;                  // softmax warps
constexpr int kMmaWarp = 8, kCopyWarp = 9, kFixWarp = 10; // and 11
constexpr int kConvWarp = 10, kConv = 6; // codes: 10-15 convert
__host__ __device__ constexpr int threads_of(int bits) { return bits == 16 ? 384 : 512; }
// K and V tiles in flight
__host__ __device__ constexpr int stages_of(int bits) { return bits == 16 ? 5 : 4; }
constexpr int kPanel = 16384;             // 128 rows x 64 channels
constexpr long long kWait = 2000000000LL; // ~1 s
constexpr float kLazy = 8.0f;
// f16 weights are formed times 2^kBoost: a reference may lag by 2^kLazy, so they stay below
// 2^15, and what f16's least step leaves of a small one is 2^-32 of the row's largest.
constexpr int kBoost = 7;
constexpr float kFar = 16777216.0f;      // 2^24: no bits below 1
constexpr int kPolyPairs = 1;             // of every four pairs of weights, on the FMA pipe
// registers of a softmax thread and of the others
__host__ __device__ constexpr int soft_regs(int bits) { return bits == 16 ? 200 : 144; }
__host__ __device__ constexpr int role_regs(int bits) { return bits == 16 ? 96 : 112; }
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS = 0, kColO = 256; // + 128 for B

__device__ __forceinline__ uint32_t su32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *b, uint32_t n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t *b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(b)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t *b, uint32_t par) {
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(su32(b)), "r"(par)
                 : "memory");
    return done != 0;
}
// Bounded wait of a whole warp, one verdict for all its lanes; on timeout the
// handle's status records it.
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t par, unsigned int *status) {
    bool ok = bar_try(b, par);
    if (!ok) {
        const long long t0 = clock64();
        while (!(ok = bar_try(b, par)))
            if (clock64() - t0 > kWait) {
                atomicOr(status, kPagesGaveUp);
                break;
            }
    }
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptor, 128-byte swizzle (layout 2), version 1.
// K-major: sbo = 1024 between groups of 8 rows.  MN-major: sbo = 1024 between
// groups of 8 tokens, lbo = one 64-channel panel.
__device__ __forceinline__ uint64_t sdesc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16: fp32 D, A and B of one type (1 = bf16), A K-major
__device__ __forceinline__ uint32_t idesc(int bf16, int N, int b_mn_major) {
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)b_mn_major << 16) |
           ((uint32_t)(N >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
}

// One asm block per step of the issuing warp: one elect.sync, the MMAs by the
// elected lane, and the commits that publish them (a commit arrives on its barrier
// when every MMA issued before it has completed).
#define KIVI_SS(off) \
    "add.u64 a, %1, " #off ";\n\tadd.u64 b, %2, " #off ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, t;\n\t"
#define KIVI_COMMIT(bar) "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [" bar "];\n\t"
// S = Q K^T over D channels: 32 bytes a step within a 64-channel panel, panels
// kPanel bytes apart; publishes S on `done` and, if release, K's stage on `freed`.
template <int D>
__device__ __forceinline__ void mma_qk(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint64_t *done, uint64_t *freed,
                                       bool release) {
#define KIVI_QK(steps)                                                                                   \
    asm volatile("{\n\t.reg .pred p, e, t, r;\n\t.reg .b64 a, b;\n\telect.sync _|e, 0xffffffff;\n\t"      \
                 "setp.ne.b32 p, %4, %4;\n\tsetp.eq.b32 t, %4, %4;\n\tsetp.ne.and.b32 r, %6, 0, e;\n\t"    \
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t" steps                  \
                 "@e " KIVI_COMMIT("%4") "@r " KIVI_COMMIT("%5") "}" ::"r"(d),                            \
                 "l"(a), "l"(b), "r"(id), "r"(su32(done)), "r"(su32(freed)), "r"((uint32_t)release)       \
                 : "memory")
    static_assert(kPanel / 16 == 1024, "panel offset below");
    if constexpr (D == 32) KIVI_QK(KIVI_SS(2));
    else if constexpr (D == 64) KIVI_QK(KIVI_SS(2) KIVI_SS(4) KIVI_SS(6));
    else if constexpr (D == 96) KIVI_QK(KIVI_SS(2) KIVI_SS(4) KIVI_SS(6) KIVI_SS(1024) KIVI_SS(1026));
    else KIVI_QK(KIVI_SS(2) KIVI_SS(4) KIVI_SS(6) KIVI_SS(1024) KIVI_SS(1026) KIVI_SS(1028) KIVI_SS(1030));
#undef KIVI_QK
}
// O += P V over 64 tokens: 4 steps, P 8 columns and V 2048 bytes a step.
#define KIVI_TS(i) \
    "add.u32 a, %1, 8 * " #i ";\n\tadd.u64 b, %2, 128 * " #i ";\n\t@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, t;\n\t"
__device__ __forceinline__ void mma_pv(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint64_t *freed, bool release) {
    asm volatile("{\n\t.reg .pred e, t, r;\n\t.reg .b32 a;\n\t.reg .b64 b;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "setp.eq.b32 t, %4, %4;\n\tsetp.ne.and.b32 r, %5, 0, e;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, t;\n\t" KIVI_TS(1) KIVI_TS(2) KIVI_TS(3)
                 "@r " KIVI_COMMIT("%4") "}" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(su32(freed)), "r"((uint32_t)release)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *b) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e " KIVI_COMMIT("%0") "}" ::"r"(su32(b)) : "memory");
}
#undef KIVI_SS
#undef KIVI_TS
#undef KIVI_COMMIT
__device__ __forceinline__ void copy_box(void *dst, const CUtensorMap *map, int x, int y, uint64_t *b) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
                 "[%4];" ::"r"(su32(dst)),
                 "l"(map), "r"(x), "r"(y), "r"(su32(b))
                 : "memory");
}

// 16 consecutive 32-bit columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float *v) {
    uint32_t r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
                 "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {"
                 "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// 64 consecutive 32-bit columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float *v) {
    uint32_t r[64];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
                 "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
                 "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
                 "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                   "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                   "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                   "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
// 32 consecutive 32-bit columns of this thread's tensor-memory lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
    uint32_t r[32];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
                 "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
                 "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                 "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                 "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                 "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

// 2^x (relative error 2^-22, -inf -> 0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// NaN if any is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// (a0, a1) * m + c, one instruction
__device__ __forceinline__ void fma2s(float &a0, float &a1, float m, float c) {
    asm("{\n\t.reg .b64 ra, rm, rc;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rm, {%2, %2};\n\tmov.b64 rc, {%3, %3};\n\t"
        "fma.rn.f32x2 ra, ra, rm, rc;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(m), "f"(c));
}
__device__ __forceinline__ void add2(float &a0, float &a1, float b0, float b1) {
    asm("{\n\t.reg .b64 ra, rb;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rb, {%2, %3};\n\tadd.rn.f32x2 ra, ra, rb;\n\t"
        "mov.b64 {%0, %1}, ra;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(b0), "f"(b1));
}
__device__ __forceinline__ void fma2c(float &a0, float &a1, float x0, float x1, float c) { // a = a * x + c
    asm("{\n\t.reg .b64 ra, rx, rc;\n\tmov.b64 ra, {%0, %1};\n\tmov.b64 rx, {%2, %3};\n\tmov.b64 rc, {%4, %4};\n\t"
        "fma.rn.f32x2 ra, ra, rx, rc;\n\tmov.b64 {%0, %1}, ra;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(x0), "f"(x1), "f"(c));
}
// 2^x of a pair on the FMA pipe, for x below 2^6: x = n + f with n an integer and
// |f| <= 1/2, 2^f by a polynomial of degree 4 that is 1 at 0 (fitted for the least
// relative error under that: 2.9e-6), n added to its exponent.  So 2^-127, where x ends,
// comes out as 0: the weight of a hidden score is 0, and a large finite value meets no
// row that does not see it.  Between -126 and -127 results lie below 2^-126.  The special
// function unit's 16 results a cycle would take as long for a tile as the tensor
// pipe does, so some of the tile's weights come from here.
__device__ __forceinline__ void ex2_pair(float &x0, float &x1) {
    constexpr float magic = 12582912.0f; // 1.5 * 2^23: adding it leaves round(x) in the low bits
    x0 = fmaxf(x0, -127.0f), x1 = fmaxf(x1, -127.0f);
    float t0 = x0, t1 = x1;
    add2(t0, t1, magic, magic);
    float r0 = t0, r1 = t1;
    add2(r0, r1, -magic, -magic);
    asm("{\n\t.reg .b64 rx, rr, rm;\n\tmov.b64 rx, {%0, %1};\n\tmov.b64 rr, {%2, %3};\n\tmov.b64 rm, {%4, %4};\n\t"
        "fma.rn.f32x2 rx, rr, rm, rx;\n\tmov.b64 {%0, %1}, rx;\n\t}" // f = x - n
        : "+f"(x0), "+f"(x1)
        : "f"(r0), "f"(r1), "f"(-1.0f));
    float p0 = 0.009582576341927052f, p1 = p0;
    fma2c(p0, p1, x0, x1, 0.05590682849287987f);
    fma2c(p0, p1, x0, x1, 0.24024106562137604f);
    fma2c(p0, p1, x0, x1, 0.6931241154670715f);
    fma2c(p0, p1, x0, x1, 1.0f);
    x0 = __uint_as_float(__float_as_uint(p0) + (__float_as_uint(t0) << 23));
    x1 = __uint_as_float(__float_as_uint(p1) + (__float_as_uint(t1) << 23));
}
template <bool F16> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}
__device__ __forceinline__ uint32_t pack_out(bool f16, float a, float b) { return f16 ? pack2<true>(a, b) : pack2<false>(a, b); }
__device__ __forceinline__ float unpack(bool f16, uint16_t x) {
    return f16 ? __half2float(__ushort_as_half(x)) : __uint_as_float((uint32_t)x << 16);
}

// ---------------------------------------------------------------- the flat list

// One block of one sequence: its rows, what they see, its cached tiles (the
// first `ns` hold first tokens, then come tiles ws ..).
struct Block {
    int b, i0, ntok;       // sequence, first new token and number of them
    int start, n, kv;      // the sequence's span
    int p0, p1;            // positions of the first and last token
    int lo, ns, ws, nt;
};
// The token at which the window that ends with position p starts, where there is a window
// (negative: with the first token; p may lie that far before it that p - window + 1 does
// not fit 32 bits).
__device__ __forceinline__ int window_start(const PagesAttn &a, int p) { return max(p, -1) - a.window + 1; }
__device__ __forceinline__ Block make_block(const PagesAttn &a, int TB, int b, const Span &s, int i) {
    Block k;
    k.b = b, k.start = s.start, k.n = s.n, k.kv = s.kv;
    k.i0 = i * TB;
    k.ntok = min(TB, s.n - k.i0);
    k.p0 = s.kv - s.n + k.i0;
    k.p1 = k.p0 + k.ntok - 1;
    k.lo = a.window ? max(0, window_start(a, k.p0)) : 0;
    k.ws = k.lo / kTok;
    k.ns = min((min(a.sinks, k.lo) + kTok - 1) / kTok, k.ws);
    // rows that see nothing still need a tile: it writes their zeros
    k.nt = max(1, k.ns + max(0, (k.p1 >= 0 ? k.p1 / kTok + 1 : 0) - k.ws));
    return k;
}
__device__ __forceinline__ int blocks_of(int n, int TB) { return (n + TB - 1) / TB; }

// Each (block, head) takes kSegCost entries of the list before its tiles: what
// starting and ending it costs, in tiles' time, so that runs of short blocks are no
// longer than others.
constexpr int kSegCost = 4;
__device__ __forceinline__ int entries(const Block &k) { return k.nt + kSegCost; }

// A CTA's run of the list, walked by its copy warp.
struct Walk {
    long long f, end, row0; // entries of the flat list; first entry of the current (block, head)
    int i, h;               // block of the sequence, head
    Block k;
};
// One (block, head)'s part in a CTA, as the copy warp publishes it to the others.
struct Seg {
    Block k;
    int t0, n;          // its tiles t0 .. t0 + n - 1; n == 0 ends the run
    int h, rows;        // kv head, query rows
    int dual;           // one row tile: A takes even tiles, B odd ones
    int nA, nB;         // tiles of each
    int whole, c0, c1;  // no other CTA has a part; else the CTAs that do
    int part;           // this CTA's part among the parts of all
    uint32_t item, edges; // copies and edge tiles of the run before it
};
// False where the run holds none of the (block, head)'s tiles.
__device__ __forceinline__ bool make_seg(const PagesAttn &a, const Walk &w, long long begin, long long per, Seg &s) {
    const long long tile0 = w.row0 + kSegCost; // entry of its first tile
    s.k = w.k;
    s.t0 = (int)max(0ll, w.f - tile0);
    s.n = (int)max(0ll, min((long long)w.k.nt, w.end - tile0)) - s.t0;
    if (s.n <= 0) return false;
    s.h = w.h;
    s.rows = w.k.ntok * a.G;
    s.dual = s.rows <= kRows;
    if (s.dual) {
        s.nA = (s.n + 1) / 2, s.nB = s.n / 2;
    } else {
        // A's last row sees no tile past its own
        const int pA = w.k.p0 + (kRows - 1) / a.G;
        const int tA = max(1, w.k.ns + max(0, (pA >= 0 ? pA / kTok + 1 : 0) - w.k.ws));
        s.nA = max(0, min(tA - s.t0, s.n)), s.nB = s.n;
    }
    const bool first = tile0 >= begin; // its first tile is in this CTA
    s.whole = first && tile0 + w.k.nt <= begin + per;
    s.c0 = s.c1 = s.part = 0;
    if (!s.whole) {
        s.c0 = (int)(tile0 / per), s.c1 = (int)((tile0 + w.k.nt - 1) / per);
        s.part = 2 * blockIdx.x + (first ? 1 : 0);
    }
    return true;
}
__device__ __forceinline__ bool walk_next(const PagesAttn &a, int TB, Walk &w) {
    w.f = w.row0 + entries(w.k);
    if (w.f >= w.end) return false;
    w.row0 = w.f;
    if (++w.h < a.st.H) return true;
    w.h = 0;
    Span sp{w.k.start, w.k.n, w.k.kv};
    int b = w.k.b;
    if (++w.i >= blocks_of(w.k.n, TB)) {
        w.i = 0;
        do {
            sp = pages_span(a.b, a.st, ++b);
        } while (sp.n == 0);
    }
    w.k = make_block(a, TB, b, sp, w.i);
    return true;
}
__device__ __forceinline__ int tile_token(const Block &k, int t) { return (t < k.ns ? t : t - k.ns + k.ws) * kTok; }
// Some row of the block does not see some token of the tile.
__device__ __forceinline__ bool tile_edge(const PagesAttn &a, const Block &k, int T) {
    if (T + kTok - 1 > k.p0) return true;
    return a.window && T < window_start(a, k.p1) && T + kTok > a.sinks;
}
// The same of one segment's tiles, from registers.
struct Tiles {
    int t0, ns, skip, p0, low, sinks;
    __device__ __forceinline__ Tiles(const PagesAttn &a, const Seg &s)
        : t0(s.t0), ns(s.k.ns), skip((s.k.ws - s.k.ns) * kTok), p0(s.k.p0), low(a.window ? window_start(a, s.k.p1) : 0),
          sinks(a.sinks) {}
    __device__ __forceinline__ int token(int j) const { return (t0 + j) * kTok + (t0 + j < ns ? 0 : skip); }
    __device__ __forceinline__ bool edge(int T) const { return T + kTok - 1 > p0 || (T < low && T + kTok > sinks); }
};
// Some row of the block sees token t.
__device__ __forceinline__ bool token_seen(const PagesAttn &a, const Block &k, int t) {
    return t <= k.p1 && (t >= k.lo || t < a.sinks);
}

constexpr int kSegs = 4;     // segments published ahead
// warps that read them: softmax, MMA, and those that touch the operand tiles
__host__ __device__ constexpr int readers_of(int bits) { return kSoft + 1 + (bits == 16 ? 2 : kConv); }
struct Shared {
    uint64_t full[5], empty[5]; // stages_of(bits) in use
    uint64_t seg_full[kSegs], seg_empty[kSegs];
    uint64_t q_full[2], s_full[2], h_full[2], p_full[2], o_full[2]; // h: the first half of P
    uint64_t edge[4], half[4]; // an edge tile's V has landed, is half through
    uint64_t meet;             // the softmax warps
    uint64_t range[4], conv;   // codes: a tile's exponents are known; the converting warps
    uint64_t drain;
    uint32_t flags[4][4]; // 16-bit pages: tokens of an edge tile whose value row is not finite
    uint32_t tmem;
    int last;
    long long scan[16];
    Walk walk;
    Seg seg[kSegs];
    PagesAttn args; // for the functions out of line: the parameters' own place is slow to read by address
};

// Codes: the operands are f16, a tile's keys and values times 2^-exponent (largest
// finite one below 2^14; of the values' kKeep more are left free rather than O moved),
// a row's query likewise, and a token's (scale, centre).  The largest token may be one that
// some rows do not see, or that weighs nothing, so tokens 2^kSpan apart do not share an
// exponent: the tile's is that of its largest token, or of the largest outside that one's 32
// if it is as far below, and tokens above it or 2^kSpan below stand apart.  Their keys get
// exponents of their own, undone in their columns of S, and their values are added apart.
constexpr int kKeep = 6, kSpan = 12, kOdd = 1024;
struct SharedCodes {
    int kexp[4], vexp[4];  // of tile counter & 3, as far as lift; kOdd more where tokens stand apart
    uint32_t apart[4][4];  // tokens whose values are added apart
    int16_t lift[4][kTok]; // how far the exponents of keys with one of their own lie above the tile's
    float4 range[2][4];    // largest key and value, smallest but 0 of both (values: -1 if some are not finite), per warp, by tile parity
    float4 token[2][kTok]; // key scale, key centre, value scale, value centre
    int qexp[2 * kRows];
};
constexpr int smem_bytes(int bits, int np) {
    return (2 + stages_of(bits)) * np * kPanel + (int)sizeof(Shared) + (bits == 16 ? 0 : (int)sizeof(SharedCodes)) + 1024;
}
static_assert(smem_bytes(16, 2) <= 232448 && smem_bytes(8, 2) <= 232448, "shared memory per block");

__device__ __forceinline__ float exp2i(int k) { return __uint_as_float((uint32_t)(max(-126, min(127, k)) + 127) << 23); }
// e with x 2^-e < 2^14 for x >= 0 (the upper end of f16, so that what is far smaller
// than x keeps its bits too); -126 at least
__device__ __forceinline__ int f16_exponent(float x) { return max(-126, (int)(__float_as_uint(x) >> 23) - 140); }
// c 2^e, a score's exp2 units, for e between -252 and 230: positive and finite where c is
// a number, since a hidden score is -inf and the scores of zero queries or keys (whose
// exponents are the least there are) are 0, and neither may become NaN by it.
__device__ __forceinline__ float score_units(float c, int e) {
    const int h = e >> 1;
    float y = c * __uint_as_float((uint32_t)(h + 127) << 23) * __uint_as_float((uint32_t)(e - h + 127) << 23);
    asm("max.NaN.f32 %0, %0, 0f00800000;" : "+f"(y)); // 2^-126
    asm("min.NaN.f32 %0, %0, 0f7f7fffff;" : "+f"(y));
    return y;
}

// A tile's scores, in tensor memory: hidden ones to -inf, in rows whose reference -off is
// not 0 the others to what times `crow` is their distance from it.  p, lo and sinks count
// from the tile's first token.
__device__ __forceinline__ void spread_scores(uint32_t cS, float crow, float off, int p, int lo, int sinks) {
#pragma unroll 1
    for (int c = 0; c < kTok; c += 16) {
        float x[16];
        tmem_ld16(cS + c, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (off != 0.0f) x[i] = __fadd_rn(__fmul_rn(x[i], crow), off) / crow;
            if (c + i > p || (c + i < lo && c + i >= sinks)) x[i] = -INFINITY;
        }
        tmem_st16(cS + c, reinterpret_cast<const uint32_t *>(x));
    }
    st_wait();
}

// A tile's weights times 2^k, where O could not go to its values' exponent.
__device__ __noinline__ void scale_weights(uint32_t cS, int k) {
    const __half2 f = __float2half2_rn(exp2i(k));
    st_wait();
#pragma unroll 1
    for (int c = 0; c < kTok / 2; c += 16) {
        float w[16];
        tmem_ld16(cS + c, w);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            __half2 *h = reinterpret_cast<__half2 *>(w + i);
            *h = __hmul2(*h, f);
        }
        tmem_st16(cS + c, reinterpret_cast<const uint32_t *>(w));
    }
}

// O and its exponents (one a row) go to a tile's values' exponent e, or, where O would
// leave fp32's range by that, as near as it can: the new exponents.
template <int ND> __device__ __noinline__ int move_exponent(uint32_t cO, int eref, int e) {
    uint32_t most = 0;
    if (__any_sync(0xffffffffu, e < eref)) {
#pragma unroll 1
        for (int c = 0; c < 32 * ND; c += 16) {
            float o[16];
            tmem_ld16(cO + c, o);
#pragma unroll
            for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(fabsf(o[i])));
        }
    }
    int n = e;
    if (e < eref && most > 0 && most < 0x7f800000u) n = min(max(e, eref + (int)(most >> 23) - 227), eref); // below 2^101
    const int d = eref - n, h = d >> 1;
    const float f0 = exp2i(h), f1 = exp2i(d - h);
#pragma unroll 1
    for (int c = 0; c < 32 * ND; c += 16) {
        float o[16];
        tmem_ld16(cO + c, o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= f0, o[i] *= f1;
        tmem_st16(cO + c, reinterpret_cast<const uint32_t *>(o));
    }
    st_wait();
    return n;
}

// 16-bit pages: rows of V that are not finite were taken out of an edge tile (flags, one
// bit per token); they are added here to the rows that see them: p > 0, so p v is v.
template <int ND, bool F16>
__device__ __noinline__ void add_unfinite(const PagesAttn &a, const uint32_t *flags, int b, int h, int T, int p, int lo,
                                          uint32_t cO) {
    for (int f = 0; f < 4; ++f) {
        uint32_t bits = flags[f];
        while (bits) {
            const int t = T + 32 * f + __ffs((int)bits) - 1;
            bits &= bits - 1;
            const bool see = t <= p && (t >= lo || t < a.sinks);
            const int64_t r = pages_row(a.st, max(pages_page(a.b, a.st, b, t), 0), h, t);
            const uint16_t *v = reinterpret_cast<const uint16_t *>(a.st.v + r * a.st.row_bytes);
#pragma unroll 1
            for (int c = 0; c < 32 * ND; c += 32) {
                float o[32];
                tmem_ld32(cO + c, o);
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float y = unpack(F16, v[c + i]);
                    if (see && !isfinite(y)) o[i] += y;
                }
                tmem_st32(cO + c, reinterpret_cast<const uint32_t *>(o));
                st_wait();
            }
        }
    }
}

// Codes: a tile of which some tokens stand apart, before its softmax.  Scores of keys with
// exponents of their own, in tensor memory, times 2^lift (finite ones stay it); then the
// row's reference, sum and O; then the values that were left out, to the rows that see them,
// with the weights of their scores (not finite ones as they are, since p > 0), O's exponent
// raised where one would not fit.
struct RowState {
    float m, l;
    int eref;
};
template <int BITS, int ND>
__device__ __noinline__ RowState settle_apart(const PagesAttn &a, const SharedCodes &sc, const Seg &s, uint32_t tile, int T, int p,
                                              int lo, uint32_t cS, float crow, RowState row) {
    const uint32_t cO = cS + (kColO - kColS);
    const int16_t *lift = sc.lift[tile & 3];
    const uint32_t *apart = sc.apart[tile & 3];
    auto see = [&](int t) { return t <= p && (t >= lo || t < a.sinks); };
    float mx = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kTok; c += 16) {
        float x[16];
        tmem_ld16(cS + c, x);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if (const int k = lift[c + i]; k != 0 && isfinite(x[i])) {
                const int h = k >> 1;
                x[i] = fminf(fmaxf(x[i] * exp2i(h) * exp2i(k - h), -3e38f), 3e38f);
            }
            if (see(T + c + i)) mx = max3(mx, x[i] * crow, mx);
        }
        tmem_st16(cS + c, reinterpret_cast<const uint32_t *>(x));
    }
    st_wait();
    const bool need = !(mx <= row.m + kLazy), move = need && row.m != -INFINITY;
    float scale = move ? ex2(row.m - mx) : 1.0f;
    row.l *= scale;
    if (need) row.m = fmaf(mx, 0.0f, mx);
    const float ref = row.m == -INFINITY ? 0.0f : row.m;
#pragma unroll 1
    for (int i = -1; i < kTok; ++i) { // (first the rescaling alone)
        if (i >= 0 && !(apart[i / 32] >> (i & 31) & 1u)) continue;
        const int t = T + max(i, 0);
        const bool add = i >= 0 && see(t);
        const int64_t r = i < 0 ? 0 : pages_row(a.st, max(pages_page(a.b, a.st, s.k.b, t), 0), s.h, t);
        const unsigned char *v = a.st.v + r * a.st.row_bytes;
        const float2 q = __ldg(a.st.vp + r);
        float x[16], w = 0.0f;
        tmem_ld16(cS + (max(i, 0) & ~15), x);
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (k == (i & 15) && add) w = ex2(__fsub_rn(__fmul_rn(x[k], crow), ref) + kBoost);
        const float most = fmaxf(fabsf(q.y), fabsf(fmaf((float)((1 << BITS) - 1), q.x, q.y)));
        int e = row.eref;
        if (w > 0.0f && isfinite(most)) e = max(e, f16_exponent(most) - 60);
        const int h = (row.eref - e) >> 1, u = -e >> 1;
        const float move1 = scale * exp2i(h), move2 = exp2i(row.eref - e - h), unit1 = exp2i(u), unit2 = exp2i(-e - u);
        row.eref = e, scale = 1.0f;
#pragma unroll 1
        for (int c = 0; c < 32 * ND; c += 16) {
            float o[16];
            tmem_ld16(cO + c, o);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int n = c + k;
                const float code = BITS == 8 ? (float)v[n] : (float)(v[n / 2] >> (4 * (n & 1)) & 15);
                const float y = fmaf(code, q.x, q.y);
                o[k] = o[k] * move1 * move2;
                if (add && (w > 0.0f || !isfinite(y))) o[k] += isfinite(y) ? w * (y * unit1 * unit2) : y;
            }
            tmem_st16(cO + c, reinterpret_cast<const uint32_t *>(o));
            st_wait();
        }
    }
    return row;
}

// Floats of one part: [D / 4][256 rows] float4 of O, then [256 rows] (m, l).
__host__ __device__ constexpr int64_t kPartFloats(int D) { return (int64_t)2 * kRows * (D + 2); }

// The last CTA of a (block, head) joins its parts, in CTA order.  A thread takes
// (row, four channels) four at a time, one step's loads independent of one
// another; eight lanes share a row, so outputs leave in runs of 64 bytes.
template <int ND> __device__ __noinline__ void join_parts(const PagesAttn &a, const Seg &s) {
    constexpr int D = 32 * ND, N = 8;
    const int G = a.G, n = (s.rows + 3) / 4 * 4 * (D / 4), tid = threadIdx.x;
    const bool f16 = a.dtype == kF16;
    // item i: groups of 8 channels-of-four x 4 rows
    for (int i0 = tid; i0 < n; i0 += 256 * N) {
        float4 acc[N];
        float mm[N], ll[N];
        int row[N], c4[N];
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int i = min(i0 + 256 * u, n - 1), g = i / 32; // 32 items: one warp's
            row[u] = g / ND * 4 + (i % 32) / 8;
            c4[u] = g % ND * 8 + i % 8;
            acc[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), mm[u] = -INFINITY, ll[u] = 0.0f;
        }
#pragma unroll 2
        for (int x = s.c0; x <= s.c1; ++x) {
            const float *px = a.part + ((int64_t)x * 2 + (x == s.c0 ? 1 : 0)) * kPartFloats(D);
            float4 y[N];
            float2 ml[N];
#pragma unroll
            for (int u = 0; u < N; ++u) {
                y[u] = __ldcg(reinterpret_cast<const float4 *>(px) + c4[u] * (2 * kRows) + row[u]);
                ml[u] = __ldcg(reinterpret_cast<const float2 *>(px + (int64_t)D * 2 * kRows) + row[u]);
            }
#pragma unroll
            for (int u = 0; u < N; ++u) {
                const float nm = fmaxf(mm[u], ml[u].x), ref = nm == -INFINITY ? 0.0f : nm;
                const float f0 = ex2(mm[u] - ref), f1 = ex2(ml[u].x - ref);
                mm[u] = nm;
                ll[u] = ll[u] * f0 + ml[u].y * f1;
                acc[u].x = acc[u].x * f0 + y[u].x * f1, acc[u].y = acc[u].y * f0 + y[u].y * f1;
                acc[u].z = acc[u].z * f0 + y[u].z * f1, acc[u].w = acc[u].w * f0 + y[u].w * f1;
            }
        }
#pragma unroll
        for (int u = 0; u < N; ++u) {
            const int r = row[u], c = c4[u];
            if (i0 + 256 * u >= n || r >= s.rows) continue;
            const int tk = r / G, hd = r - tk * G;
            const bool sees = s.k.p0 + tk >= 0;
            const float inv = 1.0f / ll[u];
            uint2 y = make_uint2(0, 0);
            if (sees) y = make_uint2(pack_out(f16, acc[u].x * inv, acc[u].y * inv), pack_out(f16, acc[u].z * inv, acc[u].w * inv));
            const int64_t otok = s.k.start + s.k.i0 + tk;
            uint16_t *d = static_cast<uint16_t *>(a.out) + otok * a.o_token + (int64_t)(s.h * G + hd) * a.o_head + 4 * c;
            if (a.o_vec) {
                *reinterpret_cast<uint2 *>(d) = y;
            } else {
                d[0] = (uint16_t)y.x, d[1] = (uint16_t)(y.x >> 16), d[2] = (uint16_t)y.y, d[3] = (uint16_t)(y.y >> 16);
            }
            if (a.lse && c == 0)
                a.lse[otok * a.Hq + s.h * G + hd] = sees ? mm[u] * 0.6931471805599453f + logf(ll[u]) : -INFINITY;
        }
    }
}

__device__ __noinline__ uint4 load_unaligned(const uint16_t *x) {
    return make_uint4(x[0] | (uint32_t)x[1] << 16, x[2] | (uint32_t)x[3] << 16, x[4] | (uint32_t)x[5] << 16,
                      x[6] | (uint32_t)x[7] << 16);
}
__device__ __noinline__ void store_unaligned(uint16_t *x, uint4 y) {
    const uint32_t e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (uint16_t)(e[k / 2] >> (16 * (k & 1)));
}

// The warp's 32 rows of O, out: normalised to the output (through the warp's part
// of its query tile, which is free by now, so that whole rows are stored a step),
// or as a part ([channels / 4][row] float4: a step's stores are contiguous).  A's
// threads add B's O where B shared their rows.  `off`: the row's output, as load_query's.
template <int ND>
__device__ __noinline__ void store_rows(const PagesAttn &a, const Seg &s, unsigned char *tile, uint32_t cO, int row0,
                                        int r0, int64_t off, bool sees, float m, float l, float fa, float fb) {
    constexpr int D = 32 * ND;
    const int lane = threadIdx.x & 31, row = row0 + lane;
    const float inv = sees ? 1.0f / l : 0.0f;
    float4 *part = reinterpret_cast<float4 *>(a.part + (int64_t)s.part * kPartFloats(D)) + r0 + row;
    const bool whole = s.whole, dual = s.dual, f16 = a.dtype == kF16;
    if (whole) fa *= inv, fb *= inv;
#pragma unroll 1
    for (int c = 0; c < D; c += 16) {
        float o[16];
        tmem_ld16(cO + c, o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= fa;
        if (dual) {
            float o2[16];
            tmem_ld16(cO + 128 + c, o2);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = fmaf(o2[i], fb, o[i]);
        }
        if (!whole) {
            if (off >= 0) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    part[(c / 4 + i) * (2 * kRows)] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 y =
                    make_uint4(pack_out(f16, o[8 * i], o[8 * i + 1]), pack_out(f16, o[8 * i + 2], o[8 * i + 3]),
                               pack_out(f16, o[8 * i + 4], o[8 * i + 5]), pack_out(f16, o[8 * i + 6], o[8 * i + 7]));
                const int cc = c / 8 + i;
                *reinterpret_cast<uint4 *>(tile + (cc >> 3) * kPanel + row * 128 + (((cc & 7) ^ (row & 7)) << 4)) =
                    sees ? y : make_uint4(0, 0, 0, 0);
            }
        }
        __syncwarp();
    }
    if (!s.whole) {
        if (off >= 0)
            reinterpret_cast<float2 *>(a.part + (int64_t)s.part * kPartFloats(D) + (int64_t)D * 2 * kRows)[r0 + row] =
                make_float2(m, l);
        return;
    }
    if (off >= 0 && a.lse) {
        const int tok = (r0 + row) / a.G;
        a.lse[(int64_t)(s.k.start + s.k.i0 + tok) * a.Hq + s.h * a.G + (r0 + row - tok * a.G)] =
            sees ? m * 0.6931471805599453f + logf(l) : -INFINITY;
    }
    constexpr int C = D / 8, R = 32 / (C > 8 ? 16 : C > 4 ? 8 : 4), L = 32 / R;
    const int c = lane % L, sub = lane / L;
    uint16_t *out = static_cast<uint16_t *>(a.out) + 8 * c;
#pragma unroll 2
    for (int i = 0; i < 32; i += R) {
        const int64_t d = __shfl_sync(0xffffffffu, (long long)off, i + sub);
        const int r = row0 + i + sub;
        if (d >= 0 && c < C) {
            const uint4 y = *reinterpret_cast<const uint4 *>(tile + (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) << 4));
            if (a.o_vec) *reinterpret_cast<uint4 *>(out + d) = y;
            else store_unaligned(out + d, y);
        }
    }
}

// The warp's 32 query rows into their tile (128-byte swizzle): 16 bytes a lane,
// whole rows a step (a lane reading its own row would touch 32 lines a load).
// `off` is the lane's own row, element offset from a.q, or -1 past the block.
template <int ND>
__device__ __noinline__ void load_query(const PagesAttn &a, unsigned char *tile, int row0, int64_t off) {
    constexpr int D = 32 * ND, C = D / 8, R = 32 / (C > 8 ? 16 : C > 4 ? 8 : 4); // chunks a row, rows a step
    constexpr int L = 32 / R;
    constexpr int U = 32 / R < 8 ? 32 / R : 8; // loads in flight; a short loop, since this code is rarely in the instruction cache
    const int lane = threadIdx.x & 31, c = lane % L, sub = lane / L;
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + 8 * c;
    const uint32_t flip = a.qsign < 0.0f ? 0x80008000u : 0u;
    unsigned char *dst = tile + (c >> 3) * kPanel;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += R * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t o = __shfl_sync(0xffffffffu, (long long)off, i0 + R * u + sub);
            v[u] = make_uint4(0, 0, 0, 0);
            if (o >= 0 && c < C) {
                if (a.q_vec) v[u] = __ldg(reinterpret_cast<const uint4 *>(q + o));
                else v[u] = load_unaligned(q + o);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row0 + i0 + R * u + sub;
            if (c < C)
                *reinterpret_cast<uint4 *>(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                    make_uint4(v[u].x ^ flip, v[u].y ^ flip, v[u].z ^ flip, v[u].w ^ flip);
        }
    }
}

// The same for codes: rows in f16 times 2^-exponent (exact, unless an element lies
// 2^-28 below the row's largest), exponents to `exps`.
template <int ND>
__device__ __noinline__ void load_query_scaled(const PagesAttn &a, unsigned char *tile, int *exps, int row0, int64_t off) {
    constexpr int D = 32 * ND, C = D / 8, L = C > 8 ? 16 : C > 4 ? 8 : 4, R = 32 / L;
    constexpr int U = 32 / R < 4 ? 32 / R : 4;
    const int lane = threadIdx.x & 31, c = lane % L, sub = lane / L;
    const uint16_t *q = static_cast<const uint16_t *>(a.q) + 8 * c;
    const bool f16 = a.dtype == kF16;
    unsigned char *dst = tile + (c >> 3) * kPanel;
#pragma unroll 1
    for (int i0 = 0; i0 < 32; i0 += R * U) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t o = __shfl_sync(0xffffffffu, (long long)off, i0 + R * u + sub);
            v[u] = make_uint4(0, 0, 0, 0);
            if (o >= 0 && c < C) {
                if (a.q_vec) v[u] = __ldg(reinterpret_cast<const uint4 *>(q + o));
                else v[u] = load_unaligned(q + o);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int r = row0 + i0 + R * u + sub;
            const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            float x[8], m = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                x[k] = unpack(f16, (uint16_t)(w[k / 2] >> (16 * (k & 1))));
                m = fmaxf(m, fabsf(x[k]));
            }
#pragma unroll
            for (int k = 1; k < L; k <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
            const int e = f16_exponent(m); // an infinite row stays infinite
            const float f = exp2i(-e) * a.qsign;
            if (c < C)
                *reinterpret_cast<uint4 *>(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                    make_uint4(pack2<true>(x[0] * f, x[1] * f), pack2<true>(x[2] * f, x[3] * f),
                               pack2<true>(x[4] * f, x[5] * f), pack2<true>(x[6] * f, x[7] * f));
            if (c == 0) exps[r] = e;
        }
    }
}

// 16 codes (4 or 2 words) -> f16 values fma(c, scale, zero), with centre = zero +
// 2^(BITS-1) scale and c - 2^(BITS-1) exact in fp32 (the code in the mantissa of
// 2^23, less 2^23 + 2^(BITS-1)); one rounding to f16.
template <int BITS> __device__ __forceinline__ void dequant16(const uint32_t *w, float scale, float centre, uint32_t (&o)[8]) {
    constexpr float bias = -8388608.0f - (float)(1 << (BITS - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) { // four codes
        float x[4];
        uint32_t b;
        if constexpr (BITS == 8) {
            b = w[i];
#pragma unroll
            for (int k = 0; k < 4; ++k) x[k] = __uint_as_float(__byte_perm(b, 0x4B000000u, 0x7440u | k));
        } else {
            b = w[i / 2] >> (16 * (i & 1));
            const uint32_t ev = b & 0x0f0fu, od = b >> 4 & 0x0f0fu; // codes 0, 2 and 1, 3 in bytes 0, 1
            x[0] = __uint_as_float(__byte_perm(ev, 0x4B000000u, 0x7440u)), x[1] = __uint_as_float(__byte_perm(od, 0x4B000000u, 0x7440u));
            x[2] = __uint_as_float(__byte_perm(ev, 0x4B000000u, 0x7441u)), x[3] = __uint_as_float(__byte_perm(od, 0x4B000000u, 0x7441u));
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            add2(x[k], x[k + 1], bias, bias);
            fma2s(x[k], x[k + 1], scale, centre);
            o[2 * i + k / 2] = pack2<true>(x[k], x[k + 1]);
        }
    }
}

// n low bits set (n may lie outside 0 .. 32)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

template <int BITS, int ND, bool F16>
__global__ void __launch_bounds__(threads_of(BITS), 1)
    pages_chunk_kernel(const __grid_constant__ PagesAttn a, int TB, int min_per, int *counters, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap) {
    constexpr int D = 32 * ND, NP = (ND + 1) / 2; // channels, 64-channel panels
    constexpr int kThreads = threads_of(BITS), kStages = stages_of(BITS);
    constexpr bool kCodes = BITS < 16;
    static_assert(!kCodes || F16, "codes become f16 operands");
    extern __shared__ unsigned char raw[];
    unsigned char *sm = raw + ((1024 - (su32(raw) & 1023)) & 1023);
    unsigned char *sq = sm, *ring = sm + 2 * NP * kPanel;
    Shared &sh = *reinterpret_cast<Shared *>(ring + kStages * NP * kPanel);
    SharedCodes &sc = *reinterpret_cast<SharedCodes *>(ring + kStages * NP * kPanel + sizeof(Shared)); // codes alone
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const PagesStore &st = a.st;
    const int H = st.H, G = a.G;
    unsigned int *status = st.status;
    if (tid == 0) {
        sh.args = a;
        for (int i = 0; i < kStages; ++i) bar_init(&sh.full[i], kCodes ? kConv : 1), bar_init(&sh.empty[i], 1);
        for (int x = 0; x < 2; ++x) {
            bar_init(&sh.q_full[x], 4);
            bar_init(&sh.s_full[x], 1);
            bar_init(&sh.h_full[x], 4);
            bar_init(&sh.p_full[x], 4);
            bar_init(&sh.o_full[x], 1);
        }
        for (int i = 0; i < kSegs; ++i) bar_init(&sh.seg_full[i], 1), bar_init(&sh.seg_empty[i], readers_of(BITS));
        for (int i = 0; i < 4; ++i) bar_init(&sh.edge[i], 1), bar_init(&sh.half[i], 1);
        bar_init(&sh.meet, kSoft);
        for (int i = 0; i < 4; ++i) bar_init(&sh.range[i], 1);
        bar_init(&sh.conv, kConv);
        bar_init(&sh.drain, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&sh.tmem)),
                     "n"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!kCodes && warp == kCopyWarp && lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
    }
    pdl_wait();
    pdl_trigger();

    // ---- the flat list: blocks of every sequence (prefix in shared memory), the
    // tiles of all of them, this CTA's run and the block it starts in
    int *pre = reinterpret_cast<int *>(sm); // [batch + 1], before the pipeline starts
    const int nw = kThreads / 32;
    auto scan = [&](long long v, long long &total) { // exclusive, over the CTA
        long long inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        __syncthreads();
        if (lane == 31) sh.scan[warp] = inc;
        __syncthreads();
        long long before = 0;
        total = 0;
        for (int w = 0; w < nw; ++w) {
            if (w < warp) before += sh.scan[w];
            total += sh.scan[w];
        }
        return before + inc - v;
    };
    long long items = 0, sum;
    for (int b0 = 0; b0 < a.b.batch; b0 += kThreads) {
        const int b = b0 + tid;
        const int n = b < a.b.batch ? blocks_of(pages_span(a.b, st, b).n, TB) : 0;
        const long long at = items + scan(n, sum);
        if (b < a.b.batch) pre[b] = (int)at;
        items += sum;
    }
    if (tid == 0) pre[a.b.batch] = (int)items;
    __syncthreads();
    auto block_at = [&](int k, int &i) { // item k: its sequence and block
        int lo = 0, hi = a.b.batch; // pre[lo] <= k < pre[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (pre[mid] <= k) lo = mid;
            else hi = mid;
        }
        i = k - pre[lo];
        return make_block(a, TB, lo, pages_span(a.b, st, lo), i);
    };
    long long tiles = 0;
    int bi;
    for (int k0 = 0; k0 < items; k0 += kThreads) {
        const int k = k0 + tid;
        scan(k < items ? entries(block_at(k, bi)) : 0, sum);
        tiles += sum;
    }
    tiles *= H;
    const long long per = max((tiles + gridDim.x - 1) / gridDim.x, (long long)min_per);
    const long long begin = per * blockIdx.x, end = min(tiles, begin + per);
    if (begin < end) {
        long long run = 0;
        for (int k0 = 0; k0 < items && run <= begin; k0 += kThreads) {
            const int k = k0 + tid;
            Block blk{};
            if (k < items) blk = block_at(k, bi);
            const long long nt = k < items ? (long long)entries(blk) * H : 0;
            const long long first = run + scan(nt, sum);
            if (nt > 0 && begin >= first && begin < first + nt) {
                Walk w;
                w.f = begin, w.end = end;
                w.h = (int)((begin - first) / entries(blk));
                w.row0 = first + (long long)w.h * entries(blk);
                w.i = bi;
                w.k = blk;
                sh.walk = w;
            }
            run += sum;
        }
    }
    proxy_fence(); // the prefix's place goes to the copies
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tm = sh.tmem;
    // a role's segments, in order: s points at the next one, false at the end
    uint32_t nseg = 0;
    const Seg *sp = nullptr;
    auto next_seg = [&]() {
        if (nseg > 0) { // done with the last one
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.seg_empty[(nseg - 1) % kSegs]);
        }
        if (!warp_wait(&sh.seg_full[nseg % kSegs], (nseg / kSegs) & 1, status)) return false;
        sp = &sh.seg[nseg % kSegs];
        ++nseg;
        return sp->n > 0;
    };
    bool ok = true;

    // A softmax thread holds a row's 128 scores.  Its spills would go to L2 (shared
    // memory leaves almost no L1), so the registers move to where they are needed.
    static_assert(256 * soft_regs(BITS) + (kThreads - 256) * role_regs(BITS) <= 65536 / kThreads / 8 * 8 * kThreads, "register split");
    if (warp < kSoft)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(soft_regs(BITS)));
    else
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(role_regs(BITS)));
    if (warp < kSoft) {
        // ------------------------------------------------------------ softmax
        const int X = warp >> 2;   // A or B
        const int row = tid & 127; // tensor-memory lane
        const uint32_t lanes = tm + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t cS = lanes + kColS + 128 * X, cO = lanes + kColO + 128 * X;
        const float c2 = a.scale * 1.4426950408889634f;
        uint32_t ns = 0, no = 0, met = 0; // tiles, blocks, meetings so far
        auto meet = [&]() { // of the softmax warps
            tc_before();
            __syncwarp();
            if (lane == 0) bar_arrive(&sh.meet);
            const bool r = warp_wait(&sh.meet, met++ & 1, status);
            tc_after();
            return r;
        };
        while (ok && next_seg()) {
            const Seg &s = *sp;
            const bool dual = s.dual;
            const int nX = X ? s.nB : s.nA;
            const int r0 = X && !dual ? kRows : 0;
            const bool live = r0 + row < s.rows;
            const int tok = live ? (r0 + row) / G : 0, head = live ? r0 + row - tok * G : 0;
            const int p = live ? s.k.p0 + tok : -1;
            const int lo = a.window ? max(0, window_start(a, p)) : 0;
            const bool any = __any_sync(0xffffffffu, live);
            float m = -INFINITY, l = 0.0f;
            if (r0 < s.rows) {
                // ---- the row's query, and an empty O
                const int64_t off = live ? (int64_t)(s.k.start + s.k.i0 + tok) * a.q_token + (int64_t)(s.h * G + head) * a.q_head : -1;
                if (X && dual) {
                } else if constexpr (kCodes) {
                    load_query_scaled<ND>(sh.args, sq + X * NP * kPanel, sc.qexp + X * kRows, row & ~31, off);
                } else {
                    load_query<ND>(sh.args, sq + X * NP * kPanel, row & ~31, off);
                }
                {
                    const uint32_t z[16] = {};
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) tmem_st16(cO + c, z);
                    st_wait();
                }
                proxy_fence();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.q_full[X]);
            }
            // B's query tile is to take B's (m, l): the last segment's rows are out of it
            if (dual && !(ok = meet())) break;
            const int n = dual ? s.n : nX;
            Tiles tl(a, s);
            uint32_t edges = s.edges; // edge tiles of the run up to this one
            float crow = c2;          // a score's exp2 units
            int eref = 0;             // O's exponent
            int kref = 0;             // the keys' exponent in crow
            for (int j = 0; j < n; ++j) {
                const int T = tl.token(j);
                const bool edge = tl.edge(T);
                if (!kCodes && edge) ++edges;
                if (dual && (j & 1) != X) continue;
                if (!(ok = warp_wait(&sh.s_full[X], ns & 1, status))) break;
                ++ns;
                tc_after();
                bool late = edge; // the weights go out in one piece
                bool odd = false; // codes: tokens of the tile stand apart
                if constexpr (kCodes) {
                    const uint32_t tile = s.item / 2 + j;
                    if (!(ok = warp_wait(&sh.range[tile & 3], tile >> 2 & 1, status))) break;
                    // B has A's queries where it shares its rows, loaded before the first S
                    const bool first = j < (dual ? 2 : 1);
                    int ke = sc.kexp[tile & 3];
                    odd = ke >= kOdd / 2;
                    late |= odd;
                    if (odd) ke -= kOdd;
                    if (first || ke != kref) {
                        kref = ke;
                        crow = score_units(c2, sc.qexp[(dual ? 0 : X * kRows) + row] + ke);
                    }
                    const int e = sc.vexp[tile & 3];
                    if (first) {
                        eref = e;
                    } else if (any && __any_sync(0xffffffffu, e != eref)) {
                        eref = move_exponent<ND>(cO, eref, e);
                        late |= __any_sync(0xffffffffu, e != eref);
                    }
                }
                if (any) {
                    // The row's scores; with codes, whose converting warps take a share of the
                    // registers, the second 64 are read again for their weights.
                    float x[kCodes ? 64 : 128];
                    auto hide = [&](float *z, int base) { // of 32 tokens from base, those out of sight
                        const uint32_t see = low_bits(p + 1 - base) & (~low_bits(lo - base) | low_bits(a.sinks - base));
#pragma unroll
                        for (int i = 0; i < 32; ++i) z[i] = see >> i & 1u ? z[i] : -INFINITY;
                    };
                    float m4[4];
                    auto most = [&](const float *z) { // 32 more
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            m4[0] = max3(m4[0], z[i], z[i + 1]);
                            m4[1] = max3(m4[1], z[i + 2], z[i + 3]);
                            m4[2] = max3(m4[2], z[i + 4], z[i + 5]);
                            m4[3] = max3(m4[3], z[i + 6], z[i + 7]);
                        }
                    };
                    if (kCodes && odd) {
                        const RowState r = settle_apart<BITS, ND>(sh.args, sc, s, s.item / 2 + j, T, p, lo, cS, crow, RowState{m, l, eref});
                        m = r.m, l = r.l, eref = r.eref;
                    }
                    tmem_ld64(cS, x);
                    if (edge) hide(x, T), hide(x + 32, T + 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i) m4[i] = x[i];
                    most(x), most(x + 32);
                    if constexpr (kCodes) {
#pragma unroll
                        for (int c = 64; c < 128; c += 32) {
                            float z[32];
                            tmem_ld32(cS + c, z);
                            if (edge) hide(z, T + c);
                            most(z);
                        }
                    } else {
                        tmem_ld64(cS + 64, x + 64);
                        if (edge) hide(x + 64, T + 64), hide(x + 96, T + 96);
                        most(x + 64), most(x + 96);
                    }
                    const float mx = max3(max3(m4[0], m4[1], m4[2]), m4[3], m4[3]) * crow;
                    // a NaN score makes the reference, and with it the row, NaN; so does an
                    // infinite one (times 0), whose own weight is infinity less infinity
                    const bool need = !(mx <= m + kLazy), move = need && m != -INFINITY;
                    const float f = move ? ex2(m - mx) : 1.0f;
                    if (need) m = fmaf(mx, 0.0f, mx);
                    if (__any_sync(0xffffffffu, move)) {
                        l *= f;
                        // every O += P V of earlier tiles is complete: S of this one was issued after them
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            float o[16];
                            tmem_ld16(cO + c, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] *= f;
                            tmem_st16(cO + c, reinterpret_cast<const uint32_t *>(o));
                        }
                    }
                    float off = m == -INFINITY ? 0.0f : -m;
                    // A product is not rounded before m, which is, is taken from it: where m has
                    // no bits below 1 the row's own largest score would be far from 0, so the
                    // scores become what times crow is their rounded distance from m.
                    if (__any_sync(0xffffffffu, fabsf(off) >= kFar)) {
                        const float ref = fabsf(off) >= kFar ? off : 0.0f;
                        off -= ref;
                        if constexpr (kCodes) {
                            spread_scores(cS, crow, ref, p - T, lo - T, a.sinks - T);
                            tmem_ld64(cS, x);
                        } else if (ref != 0.0f) {
                            const float inv = 1.0f / crow;
#pragma unroll
                            for (int i = 0; i < 128; ++i) x[i] = __fmul_rn(__fadd_rn(__fmul_rn(x[i], crow), ref), inv);
                        }
                    }
                    if constexpr (F16) off += kBoost;
                    float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
#pragma unroll
                    for (int hlf = 0; hlf < 2; ++hlf) {
                        uint32_t pk[32];
                        if (kCodes && hlf) {
                            tmem_ld64(cS + 64, x);
                            if (edge) hide(x, T + 64), hide(x + 32, T + 96);
                        }
#pragma unroll
                        for (int i = 0; i < 64; i += 8) {
                            float *y = x + (kCodes ? 0 : 64 * hlf) + i;
#pragma unroll
                            for (int q = 0; q < 8; q += 2) {
                                fma2s(y[q], y[q + 1], crow, off);
                                if (q < 2 * kPolyPairs) ex2_pair(y[q], y[q + 1]);
                                else y[q] = ex2(y[q]), y[q + 1] = ex2(y[q + 1]);
                                if (q & 2) add2(a2, a3, y[q], y[q + 1]);
                                else add2(a0, a1, y[q], y[q + 1]);
                                pk[(i + q) / 2] = pack2<F16>(y[q], y[q + 1]);
                            }
                        }
                        tmem_st32(cS + 32 * hlf, pk);
                        if (hlf == 0) { // the tensor pipe starts on the first 64 tokens
                            st_wait();
                            tc_before();
                            __syncwarp();
                            // (an edge tile's V may still change, and its O)
                            if (lane == 0 && !late) bar_arrive(&sh.h_full[X]);
                        }
                    }
                    l += (a0 + a1) + (a2 + a3);
                    if (kCodes && late) { // O is not at the exponent of this tile's values
                        const int e = sc.vexp[(s.item / 2 + j) & 3];
                        if (__any_sync(0xffffffffu, e != eref)) scale_weights(cS, e - eref);
                    }
                }
                if (!kCodes && edge) { // the tile's V has been through the fixing warps
                    const uint32_t it = s.item + 2 * j + 1;
                    if (!(ok = warp_wait(&sh.full[it % kStages], (it / kStages) & 1, status))) break;
                    const uint32_t *fl = sh.flags[(edges - 1) & 3];
                    if (fl[0] | fl[1] | fl[2] | fl[3]) add_unfinite<ND, F16>(sh.args, fl, s.k.b, s.h, T, p, lo, cO);
                }
                st_wait();
                tc_before();
                __syncwarp();
                if (lane == 0) {
                    if (late || !any) bar_arrive(&sh.h_full[X]);
                    bar_arrive(&sh.p_full[X]);
                }
            }
            // ---- the rows out
            if (ok && nX > 0) ok = warp_wait(&sh.o_full[X], no++ & 1, status);
            tc_after();
            float fa = kCodes ? exp2i(eref) : 1.0f, fb = 0.0f;
            if constexpr (F16) fa *= exp2i(-kBoost), l *= exp2i(-kBoost);
            if (dual) {
                // through B's query tile, not in use here
                float2 *ml = reinterpret_cast<float2 *>(sq + NP * kPanel);
                float *fx = reinterpret_cast<float *>(ml + kRows);
                if (X) ml[row] = make_float2(m, l), fx[row] = fa;
                if (!(ok = ok && meet())) break;
                if (!X) {
                    const float2 y = ml[row];
                    const float nm = fmaxf(m, y.x), ref = nm == -INFINITY ? 0.0f : nm;
                    const float wa = ex2(m - ref), wb = ex2(y.x - ref);
                    fa *= wa, fb = fx[row] * wb;
                    m = nm;
                    l = l * wa + y.y * wb;
                }
            }
            if (!ok) break;
            if (any && !(X && dual))
                store_rows<ND>(sh.args, s, sq + X * NP * kPanel, cO, row & ~31, r0,
                                    live ? (int64_t)(s.k.start + s.k.i0 + tok) * a.o_token + (int64_t)(s.h * G + head) * a.o_head
                                         : -1,
                                    p >= 0, m, l, fa, fb);
            if (!s.whole) {
                __threadfence();
                if (!(ok = meet())) break;
                if (tid == 0) {
                    const int done = atomicAdd(counters + s.c0, 1) == s.c1 - s.c0;
                    if (done) counters[s.c0] = 0; // for the next call
                    sh.last = done;
                }
                if (!(ok = meet())) break;
                if (sh.last) {
                    __threadfence();
                    join_parts<ND>(sh.args, s);
                }
            }
            if (dual && !(ok = meet())) break; // B's O and (m, l) are read
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------------------------------------ MMA issue
        const uint32_t id_qk = idesc(!F16, kTok, 0), id_pv = idesc(!F16, D, 1);
        const uint64_t dq = sdesc(su32(sq), 16, 1024), dr = sdesc(su32(ring), 16, 1024),
                       dv = sdesc(su32(ring), kPanel, 1024);
        uint32_t np[2] = {0, 0}, nq = 0; // tiles and blocks so far, modulo 2
        auto wait = [&](uint64_t *b, uint32_t par) { return warp_wait(b, par, status); };
        // a stage of the ring and the parity of its present phase
        struct Pos {
            uint32_t slot, par;
            __device__ __forceinline__ Pos on(uint32_t n) const { // n <= kStages items on
                const bool wrap = slot + n >= kStages;
                return Pos{wrap ? slot + n - kStages : slot + n, wrap ? par ^ 1u : par};
            }
        };
        auto qk = [&](int X, int q, uint32_t slot, bool release) {
            mma_qk<D>(tm + kColS + 128 * X, dq + q * (NP * kPanel / 16), dr + slot * (NP * kPanel / 16), id_qk, &sh.s_full[X],
                      &sh.empty[slot], release);
        };
        auto pv = [&](int X, uint32_t slot, bool release) { // by halves, as the weights come
            const uint32_t o = tm + kColO + 128 * X, p = tm + kColS + 128 * X;
            const uint64_t v = dv + slot * (NP * kPanel / 16);
            if (!wait(&sh.h_full[X], np[X])) return false;
            tc_after();
            mma_pv(o, p, v, id_pv, &sh.empty[slot], false);
            if (!wait(&sh.p_full[X], np[X])) return false;
            np[X] ^= 1;
            tc_after();
            mma_pv(o, p + 32, v + 4 * 128, id_pv, &sh.empty[slot], release);
            return true;
        };
        while (ok && next_seg()) {
            const Seg &s = *sp;
            const int n = s.n, nA = s.nA;
            Pos K{s.item % kStages, s.item / kStages & 1u}; // of the tile whose O += P V is next
            ok = wait(&sh.q_full[0], nq) && wait(&sh.q_full[1], nq) && wait(&sh.full[K.slot], K.par);
            nq ^= 1;
            if (!ok) break;
            tc_after();
            if (!s.dual) {
                if (nA > 0) qk(0, 0, K.slot, false);
                qk(1, 1, K.slot, true);
                for (int i = 0; ok && i < n; ++i) {
                    const Pos V = K.on(1), N = K.on(2);
                    const bool next = i + 1 < n;
                    if (!(ok = wait(&sh.full[V.slot], V.par))) break;
                    if (i < nA && !(ok = pv(0, V.slot, false))) break;
                    if (i + 1 == nA) mma_commit(&sh.o_full[0]);
                    if (next && !(ok = wait(&sh.full[N.slot], N.par))) break;
                    if (i + 1 < nA) qk(0, 0, N.slot, false);
                    if (!(ok = pv(1, V.slot, true))) break;
                    if (next) qk(1, 1, N.slot, true);
                    K = N;
                }
                if (ok) mma_commit(&sh.o_full[1]);
            } else { // tile t is A's or B's in turn, over the one query tile
                qk(0, 0, K.slot, true);
                if (n > 1) {
                    const Pos N = K.on(2);
                    if (!(ok = wait(&sh.full[N.slot], N.par))) break;
                    qk(1, 0, N.slot, true);
                }
                for (int t = 0; ok && t < n; ++t) {
                    const int X = t & 1;
                    const Pos V = K.on(1), N = K.on(4);
                    if (!(ok = wait(&sh.full[V.slot], V.par) && pv(X, V.slot, true))) break;
                    if (t + 2 < n) {
                        if (!(ok = wait(&sh.full[N.slot], N.par))) break;
                        qk(X, 0, N.slot, true);
                    } else {
                        mma_commit(&sh.o_full[X]);
                    }
                    K = K.on(2);
                }
            }
        }
        mma_commit(&sh.drain); // tensor memory outlives every MMA
        warp_wait(&sh.drain, 0, status);
    } else if (warp == kCopyWarp) {
        // ------------------------------------------------------------ segments and copies
        Walk w = sh.walk;
        bool more = begin < end;
        const int box = min(st.page, kTok), pieces = kTok / box;
        const int piece = lane / NP, panel = lane - piece * NP; // of the lane's box; pieces * NP <= 16
        uint32_t item = 0, ne = 0;
        for (; ok; ++nseg) {
            const uint32_t slot = nseg % kSegs;
            if (nseg >= kSegs && !(ok = warp_wait(&sh.seg_empty[slot], (nseg / kSegs - 1) & 1, status))) break;
            Seg s;
            while (more && !make_seg(a, w, begin, per, s)) more = walk_next(a, TB, w);
            if (!more) s.n = 0;
            s.item = item, s.edges = ne;
            if (lane == 0) {
                sh.seg[slot] = s;
                bar_arrive(&sh.seg_full[slot]);
            }
            if (!more) break;
            const Block &k = w.k;
            for (int r = lane; r < s.rows; r += 32) { // the queries on their way to L2
                const int tok = r / G;
                const uint16_t *q = static_cast<const uint16_t *>(a.q) + (int64_t)(k.start + k.i0 + tok) * a.q_token +
                                    (int64_t)(w.h * G + r - tok * G) * a.q_head;
                asm volatile("prefetch.global.L2 [%0];" ::"l"(q) : "memory");
                if constexpr (D > 64) asm volatile("prefetch.global.L2 [%0];" ::"l"(q + 64) : "memory");
            }
            if constexpr (kCodes) { // the converting warps fetch their own
                item += 2 * s.n;
                more = walk_next(a, TB, w);
                continue;
            }
            for (int j = 0; ok && j < s.n; ++j) {
                const int T = tile_token(k, s.t0 + j), t = T + piece * box;
                // a box is needed if some row sees one of its tokens
                const bool need = piece < pieces && t <= k.p1 && (t + box > k.lo || t < a.sinks);
                int y = 0;
                if (need) y = (int)pages_row(st, max(pages_page(a.b, st, k.b, t), 0), w.h, t);
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, need)) * (uint32_t)box * 128u;
#pragma unroll
                for (int v = 0; v < 2; ++v, ++item) {
                    const uint32_t sl = item % kStages;
                    if (item >= kStages && !(ok = warp_wait(&sh.empty[sl], (item / kStages - 1) & 1, status))) break;
                    // V of an edge tile goes to the fixing warps, which then publish it
                    uint64_t *bar = v && tile_edge(a, k, T) ? &sh.edge[ne++ & 3] : &sh.full[sl];
                    if (lane == 0) bar_expect(bar, bytes);
                    __syncwarp();
                    if (need)
                        copy_box(ring + sl * (NP * kPanel) + panel * kPanel + piece * box * 128, v ? &vmap : &kmap, 64 * panel, y,
                                 bar);
                }
            }
            if (ok) more = walk_next(a, TB, w);
        }
        // no copy outlives the CTA
        for (int i = 0; !kCodes && i < kStages && (uint32_t)i < item; ++i) {
            const uint32_t it = item - 1 - i;
            warp_wait(&sh.full[it % kStages], (it / kStages) & 1, status);
        }
    } else if (kCodes && warp >= kConvWarp) {
        // ------------------------------------------------------------ codes to operand tiles
        // Of the 192 threads ct, the first 128 own a token's parameters; of the codes each
        // takes 16 channels of every RPI-th token, and fetches its next ones as it converts
        // these.
        constexpr int LP = ND > 2 ? 8 : ND == 2 ? 4 : 2, RPI = 32 * kConv / LP, N = (kTok + RPI - 1) / RPI;
        constexpr int W = BITS == 8 ? 4 : 2, ROW = D * BITS / 8;
        const int ct = tid - 32 * kConvWarp, cw = warp - kConvWarp, piece = ct % LP, sub = ct / LP;
        const bool mine = piece < 2 * ND;
        uint32_t code[N][W];
        float2 kp, vp; // parameters of token ct
        uint32_t met = 0;
        // lane i < 8: page of tokens 16 i .. of the tile, -1 where nobody sees one of them;
        // not looked at before rows_of, so that its load has time
        auto lookup = [&](const Seg &s, int T) {
            const int t = T + 16 * lane;
            const bool any = lane < 8 && t <= s.k.p1 && (t + 16 > s.k.lo || t < a.sinks);
            return any ? __ldg(a.b.table + (int64_t)s.k.b * a.b.table_stride + (t >> st.shift)) : -1;
        };
        auto rows_of = [&](const Seg &s, int T, int page) { // row number of token 16 i
            const int t = T + 16 * lane;
            const bool any = lane < 8 && t <= s.k.p1 && (t + 16 > s.k.lo || t < a.sinks);
            if (any && (unsigned)page >= (unsigned)st.num_pages) {
                atomicOr(status, kPagesBadPage);
                page = 0;
            }
            return any ? (int)pages_row(st, page, s.h, t) : -1;
        };
        // Every lane loads, from some row of the store where there is nothing to load: a
        // token that nobody sees has scale 0.
        const int shift = min(piece, 2 * ND - 1) * (2 * BITS);
        auto fetch = [&](bool v, int rows, int i) {
            const int r = sub + RPI * i, base = __shfl_sync(0xffffffffu, rows, r >> 4 & 7);
            const unsigned char *q = (v ? st.v : st.k) + (int64_t)(max(base, 0) + (r & 15)) * ROW + shift;
            if constexpr (BITS == 8)
                asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];"
                             : "=r"(code[i][0]), "=r"(code[i][1]), "=r"(code[i][2]), "=r"(code[i][W - 1])
                             : "l"(q));
            else
                asm volatile("ld.global.nc.v2.u32 {%0,%1}, [%2];" : "=r"(code[i][0]), "=r"(code[i][1]) : "l"(q));
        };
        auto params = [&](const Seg &s, int T, int rows) {
            const int base = __shfl_sync(0xffffffffu, rows, ct >> 4 & 7);
            kp = vp = make_float2(0.0f, 0.0f);
            if (ct < kTok && base >= 0 && token_seen(a, s.k, T + ct)) {
                kp = __ldg(st.kp + base + (ct & 15)), vp = __ldg(st.vp + base + (ct & 15));
            }
        };
        while (ok && next_seg()) {
            const Seg &s = *sp;
            int ve = 0; // the values' exponent
            int T = tile_token(s.k, s.t0);
            int rows = rows_of(s, T, lookup(s, T));
            params(s, T, rows);
#pragma unroll
            for (int i = 0; i < N; ++i) fetch(false, rows, i);
            for (int j = 0; ok && j < s.n; ++j) {
                const uint32_t tile = s.item / 2 + j, it = s.item + 2 * j;
                const bool edge = tile_edge(a, s.k, T), more = j + 1 < s.n;
                const int Tn = more ? tile_token(s.k, s.t0 + j + 1) : T;
                const int pagen = lookup(s, Tn);
                // ---- the tile's range: |value| <= max(|zero|, |zero + levels scale|)
                constexpr float levels = (float)((1 << BITS) - 1), half = (float)(1 << (BITS - 1));
                const float kb = fmaxf(fabsf(kp.y), fabsf(fmaf(levels, kp.x, kp.y)));
                const float vb = fmaxf(fabsf(vp.y), fabsf(fmaf(levels, vp.x, vp.y)));
                const bool kf = isfinite(kb) && isfinite(kp.x), vf = isfinite(vb) && isfinite(vp.x);
                const uint32_t km = __reduce_max_sync(0xffffffffu, kf ? __float_as_uint(kb) : 0u);
                const uint32_t vm = __reduce_max_sync(0xffffffffu, vf ? __float_as_uint(vb) : 0u);
                const uint32_t kl = __reduce_min_sync(0xffffffffu, kf && kb > 0.0f ? __float_as_uint(kb) : 0x7f7fffffu);
                const uint32_t vl = __reduce_min_sync(0xffffffffu, vf && vb > 0.0f ? __float_as_uint(vb) : 0x7f7fffffu);
                const uint32_t bad = __ballot_sync(0xffffffffu, !vf);
                if (lane == 0 && cw < 4) {
                    sc.range[tile & 1][cw] =
                        make_float4(__uint_as_float(km), __uint_as_float(vm), __uint_as_float(kl), bad ? -1.0f : __uint_as_float(vl));
                }
                if (ct < kTok)
                    sc.token[tile & 1][ct] = make_float4(kp.x, fmaf(half, kp.x, kp.y), vp.x, fmaf(half, vp.x, vp.y));
                __syncwarp();
                if (lane == 0) bar_arrive(&sh.conv);
                if (!(ok = warp_wait(&sh.conv, met++ & 1, status))) break;
                float4 g = sc.range[tile & 1][0]; // of the tile: largest, smallest but 0 (or -1)
#pragma unroll
                for (int i = 1; i < 4; ++i) {
                    const float4 x = sc.range[tile & 1][i];
                    g.x = fmaxf(g.x, x.x), g.y = fmaxf(g.y, x.y), g.z = fminf(g.z, x.z), g.w = fminf(g.w, x.w);
                }
                int ke = f16_exponent(g.x), own = f16_exponent(g.y);
                const bool split = !(g.x <= g.z * (float)(1 << kSpan) && g.y <= g.w * (float)(1 << kSpan));
                if (split) { // the largest of the other warps
                    float k2 = 0.0f, v2 = 0.0f;
                    bool ks = false, vs = false;
                    for (int i = 0; i < 4; ++i) {
                        const float4 x = sc.range[tile & 1][i];
                        if (x.x == g.x && !ks) ks = true;
                        else k2 = fmaxf(k2, x.x);
                        if (x.y == g.y && !vs) vs = true;
                        else v2 = fmaxf(v2, x.y);
                    }
                    if (k2 > 0.0f && f16_exponent(k2) < ke - kSpan) ke = f16_exponent(k2);
                    if (v2 > 0.0f && f16_exponent(v2) < own - kSpan) own = f16_exponent(v2);
                }
                // O moves when this does, so it starts with room for values four times as
                // large, and stays while they fit and lose nothing by it; zeros take any
                if (j == 0 || own > ve || (own < ve - kKeep && g.y > 0.0f)) ve = min(own + 2, 127);
                if (split) {
                    auto outside = [](float x, int e) { return x > 0.0f && (f16_exponent(x) > e || f16_exponent(x) < e - kSpan); };
                    const int lift = kf && outside(kb, ke) ? f16_exponent(kb) - ke : 0, h = -lift >> 1;
                    const bool apart = !vf || outside(vb, own);
                    const uint32_t out = __ballot_sync(0xffffffffu, apart);
                    if (ct < kTok) {
                        sc.lift[tile & 3][ct] = (int16_t)lift;
                        float4 &q = sc.token[tile & 1][ct];
                        const float f0 = exp2i(h), f1 = exp2i(-lift - h);
                        q.x = q.x * f0 * f1, q.y = q.y * f0 * f1;
                        if (apart) q.z = q.w = 0.0f;
                        if (lane == 0) sc.apart[tile & 3][cw] = out;
                    }
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.conv);
                    if (!(ok = warp_wait(&sh.conv, met++ & 1, status))) break;
                }
                if (ct == 0) {
                    sc.kexp[tile & 3] = ke + (split ? kOdd : 0), sc.vexp[tile & 3] = ve;
                    bar_arrive(&sh.range[tile & 3]);
                }
                const float kf2 = exp2i(-ke), vf2 = exp2i(-ve);
                int rowsn = -1;
#pragma unroll 1
                for (int v = 0; v < 2; ++v) {
                    const uint32_t item = it + v, slot = item % kStages;
                    if (v == 1) {
                        rowsn = rows_of(s, Tn, pagen);
                        params(s, Tn, rowsn);
                    }
                    if (item >= kStages && !(ok = warp_wait(&sh.empty[slot], (item / kStages - 1) & 1, status))) break;
                    unsigned char *dst = ring + slot * (NP * kPanel);
                    const float f = v ? vf2 : kf2;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const int r = sub + RPI * i;
                        const float4 q = sc.token[tile & 1][r & (kTok - 1)];
                        uint32_t o[8];
                        dequant16<BITS>(code[i], (v ? q.z : q.x) * f, (v ? q.w : q.y) * f, o);
                        fetch(v == 0, v ? rowsn : rows, i);
                        if (mine && r < kTok) {
                            // (the two panels' lanes store their halves in opposite order: no bank conflicts)
#pragma unroll
                            for (int u = 0; u < 2; ++u) {
                                const int e = u ^ (piece >> 2 & 1), c = 2 * piece + e;
                                *reinterpret_cast<uint4 *>(dst + (c >> 3) * kPanel + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
                                    e ? make_uint4(o[4], o[5], o[6], o[7]) : make_uint4(o[0], o[1], o[2], o[3]);
                            }
                        }
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&sh.full[slot]);
                }
                T = Tn, rows = rowsn;
            }
        }
    } else {
        // ------------------------------------------------------------ V rows of edge tiles
        while (ok && next_seg()) {
            const Seg &s = *sp;
            uint32_t ne = s.edges;
            for (int j = 0; ok && j < s.n; ++j) {
                const int T = tile_token(s.k, s.t0 + j);
                if (!tile_edge(a, s.k, T)) continue;
                const uint32_t slot = (s.item + 2 * j + 1) % kStages;
                if (!(ok = warp_wait(&sh.edge[ne & 3], (ne >> 2) & 1, status))) break;
                unsigned char *v = ring + slot * (NP * kPanel);
#pragma unroll 1
                for (int h2 = 0; h2 < 2; ++h2) {
                    const int r = 64 * (warp - kFixWarp) + 32 * h2 + lane;
                    const bool seen = token_seen(a, s.k, T + r);
                    constexpr uint32_t ex = F16 ? 0x7c00u : 0x7f80u; // all exponent bits: not finite
                    unsigned char *rowp = v + r * 128;
                    auto chunk = [&](int c) { return reinterpret_cast<uint4 *>(rowp + (c >> 3) * kPanel + (((c & 7) ^ (r & 7)) << 4)); };
                    // the row's largest magnitude pattern first; its elements one by one only
                    // where that is not finite
                    uint32_t most = 0;
#pragma unroll
                    for (int c = 0; c < D / 8; ++c) {
                        const uint4 x = *chunk(c);
                        most = __vmaxu2(most, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu),
                                                       __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
                    }
                    const bool bad = seen && ((most & 0xffffu) >= ex || (most >> 16) >= ex);
                    if (!seen) {
#pragma unroll
                        for (int c = 0; c < D / 8; ++c) *chunk(c) = make_uint4(0, 0, 0, 0);
                    } else if (bad) {
#pragma unroll 1
                        for (int c = 0; c < D / 8; ++c) {
                            uint4 x = *chunk(c);
                            uint32_t *e = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if ((e[i] & ex) == ex) e[i] &= 0xffff0000u;
                                if ((e[i] >> 16 & ex) == ex) e[i] &= 0x0000ffffu;
                            }
                            *chunk(c) = x;
                        }
                    }
                    __syncwarp();
                    const uint32_t bits = __ballot_sync(0xffffffffu, bad);
                    if (lane == 0) sh.flags[ne & 3][2 * (warp - kFixWarp) + h2] = bits;
                }
                proxy_fence();
                __syncwarp();
                if (warp != kFixWarp) {
                    if (lane == 0) bar_arrive(&sh.half[ne & 3]);
                } else {
                    ok = warp_wait(&sh.half[ne & 3], (ne >> 2) & 1, status);
                    if (ok && lane == 0) bar_arrive(&sh.full[slot]);
                }
                ++ne;
            }
        }
    }
    tc_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tm), "n"(kTmemCols) : "memory");
    }
}

template <int BITS, int ND, bool F16> cudaError_t launch_chunk(const PagesAttn &a, int sms, cudaStream_t s) {
    static std::atomic<bool> configured[64]; // calls may come from several threads
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64 || !configured[dev]) {
        e = cudaFuncSetAttribute(pages_chunk_kernel<BITS, ND, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(BITS, (ND + 1) / 2));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    int *counters = reinterpret_cast<int *>(a.part + a.part_floats) - kPagesCounters;
    const int TB = 2 * kRows / a.G;
    return launch_pdl(pages_chunk_kernel<BITS, ND, F16>, dim3((unsigned)sms), dim3(threads_of(BITS)), smem_bytes(BITS, (ND + 1) / 2), s, true, a, TB, 2,
                      counters, a.maps->k, a.maps->v);
}

template <int BITS, bool F16> cudaError_t by_dim(const PagesAttn &a, int sms, cudaStream_t s) {
    switch (a.st.D) {
    case 32: return launch_chunk<BITS, 1, F16>(a, sms, s);
    case 64: return launch_chunk<BITS, 2, F16>(a, sms, s);
    case 96: return launch_chunk<BITS, 3, F16>(a, sms, s);
    default: return launch_chunk<BITS, 4, F16>(a, sms, s);
    }
}

} // namespace

// Blocks of at least one token: up to 256 query heads per kv head.  The batch's
// prefix lies in shared memory while the list is built.
bool pages_chunk_supported(const PagesAttn &a) { return a.G <= 2 * kRows && a.b.batch <= 16384; }

int64_t pages_chunk_scratch(int sms) { return (int64_t)sms * 2 * kPartFloats(128); }

cudaError_t launch_pages_chunk(const PagesAttn &a, cudaStream_t s) {
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return e;
    if (sms > kPagesCounters || pages_chunk_scratch(sms) > a.part_floats - kPagesCounters)
        return cudaErrorInvalidConfiguration;
    ProfScope prof("pages_chunk", s);
    count_launch();
    const bool f16 = a.dtype == kF16;
    if (a.st.bits == 16) return f16 ? by_dim<16, true>(a, sms, s) : by_dim<16, false>(a, sms, s);
    return a.st.bits == 8 ? by_dim<8, true>(a, sms, s) : by_dim<4, true>(a, sms, s);
}

// Tensor maps over 16-bit pages: rows of D elements, boxes of one page's tokens
// (at most a tile's) x 64 channels, 128-byte swizzle, zeros past the last channel.
cudaError_t pages_tensor_maps(const PagesStore &st, PagesMaps *maps) {
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult found;
    cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found);
    if (e != cudaSuccess) return e;
    if (found != cudaDriverEntryPointSuccess) return cudaErrorNotSupported;
    const PFN_cuTensorMapEncodeTiled encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled>(fn);
    const cuuint64_t dims[2] = {(cuuint64_t)st.D, (cuuint64_t)st.num_pages * st.H * st.page};
    const cuuint64_t strides[1] = {(cuuint64_t)st.row_bytes};
    const cuuint32_t box[2] = {64, (cuuint32_t)std::min(st.page, kTok)}, steps[2] = {1, 1};
    const CUtensorMapDataType type = st.dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    for (int side = 0; side < 2; ++side) {
        const CUresult r = encode(side ? &maps->v : &maps->k, type, 2, side ? st.v : st.k, dims, strides, box, steps,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        if (r != CUDA_SUCCESS) return cudaErrorInvalidValue;
    }
    return cudaSuccess;
}

} // namespace kivi

// af_paged_tc.cu -- attention of chunks of new tokens over a paged KV cache on the
// tcgen05 tensor cores (af_paged_attention's path for more than a few rows per
// sequence and kv head).
//
//   S = Q K^T,  P = exp2(c S - c m),  O = sum over tiles of P V,  out = O / l
//
// c = scale * log2(e), m the row's running maximum, l the running sum of P.
//
//   * Rows: the G query heads that share a kv head see the same K and V, so the
//     rows of a work item are (token, head of the group) pairs of one sequence,
//     256 of them: two 128-row MMA tiles that share every K and V tile read.
//   * Warp 9 fetches K and V tiles of 128 positions with TMA, one box per page (and
//     64-dim panel) through the block table, into a ring of slots in the
//     128-byte-swizzled layout that the MMA reads; a page outside the pool is a
//     coordinate outside the tensor, which reads as zeros.  8-bit codes land in a
//     staging ring, and warps 12-15 turn them into FP16 slots exactly: K's codes as
//     they are, V's times their scale's power of two (kv_split_scale).  The rest of the scales is
//     applied in FP32 by the softmax, K's to the columns of S, V's (in [1, 2) for the scales that the write stores) to P
//     before its rounding: multiplied into the FP16 slots they cost a rounding
//     of every element (relative error against 64 bits of a 4096-token FP8 prompt
//     3.9e-4, 130 us; as it is 2.7e-4, 152 us; FP32 scales in shared memory 152 us).
//   * V at positions that a row does not see (behind it in its own chunk, or past the
//     end) meets weights of zero; where it is an infinity or NaN the product would be
//     NaN.  Warps 12-15 put zeros in the place of such values, and the epilogue adds
//     them back for the rows that do see them.  (K there gives scores that are
//     masked.)
//   * The output goes through shared memory (Q's place) to whole rows per half warp:
//     rows written by a thread each cost the LSU eight times the wavefronts.
//   * Warp 8 issues the MMAs.  S of both row tiles and O of both fill the 512
//     TMEM columns; P (FP16) overwrites the S it came from and is the A operand
//     of the second product straight from TMEM.  The order PV(0, j), QK(0, j+1),
//     PV(1, j), QK(1, j+1) keeps the tensor core on one row tile while the other
//     is in its softmax.
//   * Warps 0-3 and 4-7 load Q and are the softmax of row tile 0 and 1, one row per
//     thread: no shuffles.  O is rescaled only when the row's maximum has grown by more
//     than a factor 2^8 (FP8 2^7) since the last rescale (P then stays below that, exact
//     range in FP16; l and O are FP32), which ends after the first few tiles.
//   * P is rounded to FP16 for the second product, the type of V's tile: its error, at most 2^-11 of each
//     weight, is that of the FP16 output's own rounding (relative error 2.7e-4 to 2.9e-4, without it 2.1e-4).
//   * Few rows and a long cache: a work item's positions are split over the CTAs
//     of a cluster, which merge through distributed shared memory in rank order
//     -- no workspace, no second launch, the same bits every time.
//   * Bound: FP16 by the MMAs, which share shared memory's bandwidth with TMA (4 x 1024
//     new tokens over 16384, 32 heads over 8: 1131 to 1148 us in a graph, 1167 to 1175 among other calls, 906 to 942
//     TFLOP/s); 8 bits by the chain S, softmax of all columns, P V, next S in the same columns, which two row tiles do
//     not cover once the scales lengthen the softmax (4096-token FP8 prompt, 24 heads: 153 us, 674 TFLOP/s; issue
//     slots 46% used, tensor pipe 34%).
//   * Registers: 128 at launch, 184 in the softmax warps.  -Xptxas -v counts 76 to 92 bytes of spills: values that the
//     cluster's merge needs after the loop (without that part four of the six variants have none, the others 44 and
//     52).  The rest of the 152-byte frame belongs to the calls of add_mended.
//   * Every wait is bounded; one that runs out sets AF_FAULT_TC_WAIT and the
//     kernel ends without waiting further.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "af_paged.cuh"

namespace af {
namespace {

constexpr int kTile = 128;              // rows of an MMA tile; positions of a K or V tile
constexpr int kItemRows = 2 * kTile;
constexpr int kThreads = 512;
constexpr int kMmaWarp = 8, kFetchWarp = 9, kConvWarp = 12;
constexpr uint64_t kWaitNs = 2000000000ull;
constexpr int kMaxSplit = kPagedMaxSplit;
constexpr int kTmemCols = 512;

// The largest power of two of V's scale that goes into the values of a slot: its product with the largest code (-128
// among INT8's) is a finite FP16 value.
template <int FMT>
constexpr int kPowerMax = FMT == AF_KV_INT8 ? 8 : 7;

template <int FMT, int HD>
struct Shape {
    static constexpr bool kQuant = FMT != AF_KV_F16;
    static constexpr int kTileBytes = kTile * HD * 2;    // one 128 x HD FP16 tile
    static constexpr int kCodeBytes = kTile * HD;        // one 128 x HD tile of codes
    static constexpr int kSlots = HD == 64 ? 8 : kQuant ? 4 : 5;
    static constexpr int kStages = kQuant ? (HD == 64 ? 4 : 2) : 0;
    static constexpr int kQBytes = 2 * kTileBytes;
    // Scales of as many tiles: what writes tile j's has waited for the ring slot of V's tile j - 1, that is for the
    // product with V's tile j - 1 - kSlots / 2, behind the softmax that read that tile's scales.
    static constexpr int kScales = kQuant ? kSlots / 2 + 1 : 1;
    static constexpr int kRing = kQBytes, kStaging = kRing + kSlots * kTileBytes;
    static constexpr size_t kSmem = kStaging + (size_t)kStages * kCodeBytes + 1024;   // + alignment to 1 KB
    // log2 of the growth of the maximum that forces a rescale: P times the rest of any finite scale stays finite in FP16
    // (2^7 * 511.75, 2^8 * 255.9).
    static constexpr float kGrow = FMT == AF_KV_FP8_E4M3 ? 7.f : 8.f;
    // the fetch ring: slots, or staging for codes
    static constexpr int kFetch = kQuant ? kStages : kSlots;
};
static_assert(Shape<AF_KV_F16, 128>::kSmem + 2048 <= 227 * 1024 && Shape<AF_KV_INT8, 128>::kSmem + 2048 <= 227 * 1024,
              "shared memory");

struct TcArgs {
    const __half* q;
    long long q_stride;
    __half* out;
    int NH, G;
    float c;            // scale * log2(e)
    int skip_rows;      // sequences of at most this many rows (tokens x G) belong to another kernel
};

// ---- tcgen05 (PTX ISA) ----
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(ncols)
                 : "memory");
}
__device__ __forceinline__ void tmem_relinquish() {
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 or 32 consecutive 32-bit TMEM columns of this warp's 32 lanes -> registers and back.  Loaded values are there
// only after tmem_wait_ld; tmem_pin keeps their uses behind it.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_pin(uint32_t (&r)[16]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_pin(uint32_t (&r)[32]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle (layout type 2 at bits 61-63), version 1.  K-major (Q, K):
// sbo = bytes between 8-row groups.  N-major (V): lbo = bytes between 64-element panels, sbo = between 8-position
// groups.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16 instruction descriptor: FP32 accumulator, FP16 operands, A K-major, M = 128.
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool b_n_major) {
    return (1u << 4) | (b_n_major ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
}
// One box of a 5-D tensor -> shared memory, completing on an mbarrier.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int c1, int c2, int c3, int c4, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
        "[%7];" ::"r"(dst),
        "l"(map), "r"(0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// (a, b) * (m, m) + (k, k) in one packed FP32 FMA
__device__ __forceinline__ void fma2(float& a, float& b, float m, float k) {
    unsigned long long x, mm, kk;
    asm("mov.b64 %0, {%1,%2};" : "=l"(x) : "f"(a), "f"(b));
    asm("mov.b64 %0, {%1,%1};" : "=l"(mm) : "f"(m));
    asm("mov.b64 %0, {%1,%1};" : "=l"(kk) : "f"(k));
    asm("fma.rn.f32x2 %0, %0, %1, %2;" : "+l"(x) : "l"(mm), "l"(kk));
    asm("mov.b64 {%0,%1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
__device__ __forceinline__ void add2(float& a, float& b, float c, float d) {
    unsigned long long x, y;
    asm("mov.b64 %0, {%1,%2};" : "=l"(x) : "f"(a), "f"(b));
    asm("mov.b64 %0, {%1,%2};" : "=l"(y) : "f"(c), "f"(d));
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
    asm("mov.b64 {%0,%1}, %2;" : "=f"(a), "=f"(b) : "l"(x));
}
// (a, b) * (c, d) of FP32 values in one packed product
__device__ __forceinline__ void mul2(uint32_t& a, uint32_t& b, float c, float d) {
    unsigned long long x, y;
    asm("mov.b64 %0, {%1,%2};" : "=l"(x) : "r"(a), "r"(b));
    asm("mov.b64 %0, {%1,%2};" : "=l"(y) : "f"(c), "f"(d));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(y));
    asm("mov.b64 {%0,%1}, %2;" : "=r"(a), "=r"(b) : "l"(x));
}
// Eight FP16 scales of shared memory (16-byte aligned) in FP32
__device__ __forceinline__ void scales8(const __half* p, float (&f)[8]) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = x.x;
        f[2 * i + 1] = x.y;
    }
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// One lane of a converged warp, in the form from which the compiler knows that a single thread follows (the MMA's
// operands then stay in uniform registers).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}

// A row's token and head of the group, and those of every `by`-th row after it without a division each (Q's 32 rows per
// thread took 6 us with one).
struct RowOf {
    int tok, head, G, d_tok, d_head;
    __device__ __forceinline__ RowOf(int row, int g, int by) : G(g) {
        tok = row / g;
        head = row - tok * g;
        d_tok = by / g;
        d_head = by - d_tok * g;
    }
    __device__ __forceinline__ void step() {
        tok += d_tok;
        head += d_head;
        if (head >= G) {
            head -= G;
            ++tok;
        }
    }
};

struct Bars {
    uint64_t full[8], empty[8];          // ring slots
    uint64_t raw_full[4], raw_empty[4];  // staging of codes; FP16: the V tiles with masked positions (three at most)
    uint64_t s_full[2], p_full[2];       // per row tile
    uint64_t q_full[2], o_done;
};

// Bounded wait: false once the limit has passed (the fault bit is set).
__device__ __forceinline__ bool tc_wait(const uint64_t* bar, uint32_t parity, volatile int* abort, unsigned* fault) {
    const uint32_t b = smem_u32(bar);
    if (mbar_try_wait(b, parity)) return true;
    if (*abort) return false;
    if (mbar_wait_bounded(b, parity, kWaitNs)) return true;
    atomicOr(fault, (unsigned)AF_FAULT_TC_WAIT);
    *abort = 1;
    return false;
}

// Adds to a row's output (FP16, or FP32 in a cluster's part) what was taken out of V at positions [from, to).  Rare and
// out of line: the row's outputs are read back.
template <int FMT, int HD>
__device__ __noinline__ void add_mended(const Paged& p, int b, int kvh, int from, int to, __half* dst, float* part, int r,
                                        unsigned* fault) {
#pragma unroll 1
    for (int pos = from; pos < to; ++pos)
#pragma unroll 1
        for (int d = 0; d < HD; ++d) {
            const float x = v_value<FMT, HD>(p, b, pos, kvh, d, fault);
            if (fabsf(x) < INFINITY) continue;
            if (part != nullptr) part[((d >> 2) ^ (r & (HD / 4 - 1))) * 4 + (d & 3)] += x;
            else dst[d] = __float2half_rn(__half2float(dst[d]) + x);
        }
}
// The same for the chunks of a tile of codes that thread i has just converted, in rows from `from` on.
template <int HD>
__device__ __noinline__ bool mend_rows(unsigned char* tile, int i, int from) {
    constexpr int C8 = HD / 16, RC = 128 / C8;
    bool mended = false;
#pragma unroll 1
    for (int r = i / C8; r < kTile; r += RC) {
        if (r < from) continue;
#pragma unroll 1
        for (int e = 0; e < 2; ++e) {
            const int ch = 2 * (i % C8) + e;
            uint4* at = reinterpret_cast<uint4*>(tile + (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
            uint4 y = *at;
            if (mend_chunk(y)) {
                *at = y;
                mended = true;
            }
        }
    }
    return mended;
}

template <int FMT, int HD>
__global__ void __launch_bounds__(kThreads, 1) paged_chunk_kernel(const Paged p, const TcArgs a,
                                                                   const __grid_constant__ CUtensorMap k_map,
                                                                   const __grid_constant__ CUtensorMap v_map,
                                                                   unsigned* fault) {
    namespace cg = cooperative_groups;
    using Sh = Shape<FMT, HD>;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) Bars bars;
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    __shared__ volatile int s_mended;                // V had infinities or NaN where some row does not look
    __shared__ int s_item[2];                        // sequence, row tile pair
    // tiles' scales: K's, and V's without its power of two
    __shared__ __align__(16) __half s_scale[Sh::kScales][2][kTile];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int cid = blockIdx.x / S, kvh = cid % p.NKV, item = cid / p.NKV;

    pdl_launch_dependents();   // the kernel of the short sequences may begin as soon as every CTA of this one has

    // ------------------------------------------------ which work item is ours
    if (warp == 0) {
        int seen = 0, fb = -1, ft = 0;
        for (int b0 = 0; b0 < p.n_seqs && fb < 0; b0 += 32) {
            const int b = b0 + lane;
            int n = 0;
            if (b < p.n_seqs) {
                const PagedSeq s = paged_seq(p, b, fault);
                const long long rows = (long long)s.q * a.G;
                n = rows > a.skip_rows ? (int)((rows + kItemRows - 1) / kItemRows) : 0;
            }
            int inc = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += u;
            }
            const bool mine = item >= seen + inc - n && item < seen + inc;
            const unsigned who = __ballot_sync(0xffffffffu, mine);
            if (who) {
                const int src = __ffs(who) - 1;
                fb = b0 + src;
                // later rows see more positions: they go first
                ft = __shfl_sync(0xffffffffu, seen + inc - 1 - item, src);
            }
            seen += __shfl_sync(0xffffffffu, inc, 31);
        }
        if (lane == 0) {
            s_item[0] = fb;
            s_item[1] = ft;
            s_abort = 0;
            s_mended = 0;
        }
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&s_tmem), kTmemCols);
        tmem_relinquish();
    }
    if (threadIdx.x == 32) {
        for (int i = 0; i < 8; ++i) {
            mbar_init(smem_u32(&bars.full[i]), Sh::kQuant ? 128 : 1);
            mbar_init(smem_u32(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&bars.raw_full[i]), 1);
            mbar_init(smem_u32(&bars.raw_empty[i]), 128);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&bars.q_full[i]), 128);
            mbar_init(smem_u32(&bars.s_full[i]), 1);
            mbar_init(smem_u32(&bars.p_full[i]), 128);
        }
        mbar_init(smem_u32(&bars.o_done), 1);
        mbar_init_fence();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    const int b = s_item[0];
    if (b < 0) {   // no such item: the whole cluster leaves
        if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
        return;
    }
    const PagedSeq seq = paged_seq(p, b, fault);
    const int row_base = s_item[1] * kItemRows;
    const int rows = min(kItemRows, (int)min((long long)seq.q * a.G - row_base, (long long)kItemRows));
    const int n_sub = rows > kTile ? 2 : 1;          // row tiles in use
    const int ctx = seq.kv - seq.q;
    const int last_token = (row_base + rows - 1) / a.G;
    const int end = max(0, ctx + last_token + 1);    // positions any row sees
    const int tiles = (end + kTile - 1) / kTile;
    const int shift = 31 - __clz(S);                 // S is a power of two, at most 8: no division, no overflow
    const int t0 = (tiles * rank) >> shift, t1 = (tiles * (rank + 1)) >> shift;
    const int n = t1 - t0;
    // positions that every row sees; tiles from first_masked on hold others
    const int all_see = max(0, ctx + row_base / a.G + 1), first_masked = max(0, all_see / kTile - t0);
    unsigned char* q_s = smem;
    unsigned char* ring = smem + Sh::kRing;
    // the cluster merge's parts, in the buffers once they are idle: FP32 O [256][HD], then m and l [256]
    float* part_o = reinterpret_cast<float*>(smem);
    float* part_m = part_o + kItemRows * HD;
    float* part_l = part_m + kItemRows;
    static_assert((kItemRows * HD + 3 * kItemRows) * 4 <= Sh::kSmem - 1024, "parts fit");   // and the merge's factors

    auto any_abort = [&] { return __any_sync(0xffffffffu, s_abort != 0) != 0; };   // the same for the whole warp

    if (warp >= kConvWarp) {
        // --------------------------------------------------- conversion, mending
        // registers are handed over once, here, and never taken back: 2 x 184 + 56 + 88 = 4 x 128
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const int i = threadIdx.x - kConvWarp * 32;
        if (n > 0) {
            constexpr int CH = HD / 8;               // 16-byte FP16 chunks of a row
            if constexpr (!Sh::kQuant) {
                // V tiles with masked positions come by way of these warps: zeros past the end and in the place of
                // infinities and NaN
                bool mended = false;
                for (int j = first_masked; j < n; ++j) {
                    const int slot = (2 * j + 1) % Sh::kSlots;
                    tc_wait(&bars.raw_full[j - first_masked], 0, &s_abort, fault);
                    const int pos0 = (t0 + j) * kTile, from = max(0, all_see - pos0), left = end - pos0;
                    unsigned char* v = ring + slot * Sh::kTileBytes;
                    for (int x = from * CH + i; x < kTile * CH; x += 128) {
                        const int r = x / CH, ch = x % CH;
                        uint4* at = reinterpret_cast<uint4*>(v + (ch >> 3) * (kTile * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                        uint4 y = make_uint4(0u, 0u, 0u, 0u);
                        if (r < left) {
                            y = *at;
                            if (!mend_chunk(y)) continue;
                            mended = true;
                        }
                        *at = y;
                    }
                    if (mended) s_mended = 1;
                    fence_async_smem();
                    named_bar_sync(1, 128);
                    if (i == 0) mbar_arrive(smem_u32(&bars.full[slot]));
                }
            } else {
                constexpr int C8 = HD / 16;          // 16-code chunks of a row
                constexpr int RC = 128 / C8, KR = kTile / RC;
                const int c8 = i % C8, rq = i / C8;
                // code chunk c8 makes FP16 chunks 2 c8 and 2 c8 + 1 of panel c8 / 4
                const uint32_t row_at = (c8 >> 2) * (kTile * 128) + rq * 128;
                const uint32_t x0 = ((2 * c8) & 7) ^ (rq & 7), x1 = ((2 * c8 + 1) & 7) ^ (rq & 7);
                // a warp owns the rows that its threads convert: lane l row `mine`, row rq + x RC lane rq % RPW + RPW x
                constexpr int RPW = 32 / C8;
                const int mine = (i >> 5) * RPW + lane % RPW + RC * (lane / RPW);
                __half sk, sv;                       // of row `mine` of the next tile
                auto fetch = [&](int j) {
                    const int pos = (t0 + j) * kTile + mine;
                    sk = sv = __float2half_rn(0.f);
                    const int page = j < n && pos < end ? paged_page(p, b, pos, fault) : -1;
                    if (page >= 0) {
                        const long long at = paged_scale(p, page, pos, kvh);
                        sk = __ldg(p.ks + at);
                        sv = __ldg(p.vs + at);
                    }
                };
                fetch(0);
                for (int j = 0; j < n; ++j) {
                    // V's scale = power * rest, both exact; an infinity or NaN stays with the values, which are mended
                    const KvScaleParts parts = kv_split_scale<FMT, kPowerMax<FMT>>(__half2float(sv));
                    const bool odd = (__half_as_ushort(sv) & 0x7c00u) == 0x7c00u;
                    const uint32_t power = __half_as_ushort(odd ? sv : parts.power);
                    s_scale[j % Sh::kScales][0][mine] = sk;
                    s_scale[j % Sh::kScales][1][mine] = __float2half_rn(odd ? 1.f : parts.rest);
                    fetch(j + 1);
                    const int left = end - (t0 + j) * kTile;   // positions of the tile that exist
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        const int m = 2 * j + kv, slot = m % Sh::kSlots, st = m % Sh::kStages;
                        tc_wait(&bars.raw_full[st], (m / Sh::kStages) & 1, &s_abort, fault);
                        if (m >= Sh::kSlots) tc_wait(&bars.empty[slot], (m / Sh::kSlots - 1) & 1, &s_abort, fault);
                        const unsigned char* src = smem + Sh::kStaging + st * Sh::kCodeBytes + i * 16;
                        unsigned char* dst = ring + slot * Sh::kTileBytes + row_at;
#pragma unroll
                        for (int k = 0; k < KR; ++k) {
                            const int r = rq + k * RC;
                            uint4 code = *reinterpret_cast<const uint4*>(src + k * 2048);
                            if (r >= left) code = make_uint4(0u, 0u, 0u, 0u);
                            const uint32_t pw = kv == 1 ? __shfl_sync(0xffffffffu, power, rq % RPW + RPW * k) * 0x10001u : 0u;
                            const __half2 s2 = *reinterpret_cast<const __half2*>(&pw);
                            const uint32_t in[4] = {code.x, code.y, code.z, code.w};
                            uint32_t o[8];
#pragma unroll
                            for (int w = 0; w < 4; ++w) {
                                kv_unpack4<FMT>(in[w], o[2 * w], o[2 * w + 1]);
                                if (kv == 1) {
                                    o[2 * w] = mul_half2(o[2 * w], s2);
                                    o[2 * w + 1] = mul_half2(o[2 * w + 1], s2);
                                }
                            }
                            *reinterpret_cast<uint4*>(dst + k * RC * 128 + x0 * 16) = make_uint4(o[0], o[1], o[2], o[3]);
                            *reinterpret_cast<uint4*>(dst + k * RC * 128 + x1 * 16) = make_uint4(o[4], o[5], o[6], o[7]);
                        }
                        if (kv == 1 && j >= first_masked && mend_rows<HD>(dst - row_at, i, max(0, all_see - (t0 + j) * kTile)))
                            s_mended = 1;
                        fence_async_smem();
                        mbar_arrive(smem_u32(&bars.full[slot]));
                        mbar_arrive(smem_u32(&bars.raw_empty[st]));
                    }
                }
            }
        }
    } else if (warp >= kMmaWarp) {
        // ----------------------------------------------------------- MMA issue
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kMmaWarp) {
            constexpr uint32_t qk_desc = instr_desc(kTile, false), pv_desc = instr_desc(HD, true);
            const uint32_t q0 = smem_u32(q_s), r0 = smem_u32(ring);
            auto qk = [&](int i, int m) {   // S_i = Q_i K^T with the K tile of ring entry m
                const uint32_t k0 = r0 + (m % Sh::kSlots) * Sh::kTileBytes;
#pragma unroll
                for (int s = 0; s < HD / 16; ++s) {
                    const uint32_t off = (s >> 2) * (kTile * 128) + (s & 3) * 32;
                    mma_ss(tmem + i * kTile, smem_desc(q0 + i * Sh::kTileBytes + off, 16, 1024),
                           smem_desc(k0 + off, 16, 1024), qk_desc, s > 0);
                }
                tc_commit(smem_u32(&bars.s_full[i]));
            };
            auto pv = [&](int i, int m, bool acc) {   // O_i (+)= P_i V
                const uint32_t v0 = r0 + (m % Sh::kSlots) * Sh::kTileBytes;
#pragma unroll
                for (int s = 0; s < kTile / 16; ++s)
                    mma_ts(tmem + 2 * kTile + i * kTile, tmem + i * kTile + s * 8,
                           smem_desc(v0 + s * 2048, kTile * 128, 1024), pv_desc, acc || s > 0);
            };
            auto full = [&](int m) {
                tc_wait(&bars.full[m % Sh::kSlots], (m / Sh::kSlots) & 1, &s_abort, fault);
                tc_fence_after();
            };
            if (n > 0) {
                full(0);
                for (int i = 0; i < n_sub; ++i) {
                    tc_wait(&bars.q_full[i], 0, &s_abort, fault);
                    tc_fence_after();
                    if (!any_abort() && elect_one()) qk(i, 0);
                    __syncwarp();
                }
                if (!any_abort() && elect_one()) tc_commit(smem_u32(&bars.empty[0]));
                __syncwarp();
                for (int j = 0; j < n; ++j) {
                    const int mv = 2 * j + 1, mk = 2 * j + 2;
                    full(mv);
                    for (int i = 0; i < n_sub; ++i) {
                        tc_wait(&bars.p_full[i], j & 1, &s_abort, fault);
                        tc_fence_after();
                        if (!any_abort() && elect_one()) pv(i, mv, j > 0);
                        __syncwarp();
                        if (j + 1 < n) {
                            if (i == 0) full(mk);
                            if (!any_abort() && elect_one()) qk(i, mk);
                            __syncwarp();
                        }
                    }
                    if (!any_abort() && elect_one()) {
                        tc_commit(smem_u32(&bars.empty[mv % Sh::kSlots]));
                        if (j + 1 < n) tc_commit(smem_u32(&bars.empty[mk % Sh::kSlots]));
                        else tc_commit(smem_u32(&bars.o_done));
                    }
                    __syncwarp();
                }
            }
        } else if (warp == kFetchWarp) {
            // -------------------------------------------------------------- fetch
            // one box per page of the tile and, for FP16, 64-dim panel: a lane each
            constexpr int PN = Sh::kQuant ? 1 : HD / 64;
            constexpr int kRow = Sh::kQuant ? HD : 128;      // bytes of a box's row
            const int box_rows = min(1 << p.page_shift, kTile);
            const int panel = lane % PN, box = lane / PN;
            uint64_t* fetched = Sh::kQuant ? bars.raw_full : bars.full;
            uint64_t* empty = Sh::kQuant ? bars.raw_empty : bars.empty;
            const uint32_t base = smem_u32(smem + (Sh::kQuant ? Sh::kStaging : Sh::kRing)) + panel * (kTile * 128) +
                                  box * box_rows * kRow;
            int page = 0, m = 0;
            for (; m < 2 * n && !any_abort(); ++m) {
                const int st = m % Sh::kFetch, pos0 = (t0 + (m >> 1)) * kTile;
                const int boxes = (min(kTile, end - pos0) + box_rows - 1) / box_rows;   // those with positions that exist
                const int pos = pos0 + box * box_rows;
                if (!(m & 1) && box < boxes) {               // K: look the page up; V: the same
                    page = paged_page(p, b, pos, fault);
                    if (page < 0) page = max(p.n_pages, 1);  // outside the tensor: zeros
                }
                if (m >= Sh::kFetch) tc_wait(&empty[st], (m / Sh::kFetch - 1) & 1, &s_abort, fault);
                // a V tile with masked positions: warps 12-15 hand it on
                const int mask = (m & 1) && !Sh::kQuant ? (m >> 1) - first_masked : -1;
                const uint32_t bar = smem_u32(mask >= 0 ? &bars.raw_full[mask] : &fetched[st]);
                if (lane == 0) mbar_arrive_expect_tx(bar, (uint32_t)(boxes * box_rows * kRow * PN));
                __syncwarp();
                if (box < boxes)
                    tma_load(base + st * (Sh::kQuant ? Sh::kCodeBytes : Sh::kTileBytes), (m & 1) ? &v_map : &k_map,
                             paged_slot_of(pos, p.page_shift), panel, kvh, page, bar);
            }
            if (any_abort()) {   // nothing may still be landing when the CTA ends
                for (int x = max(0, m - Sh::kFetch); x < m; ++x)
                    mbar_wait_bounded(smem_u32(&fetched[x % Sh::kFetch]), (x / Sh::kFetch) & 1, kWaitNs);
                for (int x = 0; !Sh::kQuant && x < n - first_masked; ++x)
                    if (2 * (first_masked + x) + 1 < m) mbar_wait_bounded(smem_u32(&bars.raw_full[x]), 0, kWaitNs);
            }
        }
    } else {
        // ------------------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int i = warp >> 2, r = threadIdx.x & 127;   // row tile, row (= TMEM lane)
        if (n > 0 && i < n_sub) {                         // Q: this row tile
            constexpr int CH = HD / 8, RS = 128 / CH;     // 16-byte chunks of a row, rows between a thread's (a multiple of 8)
            const int c = r % CH, r0 = r / CH;
            const uint32_t at = smem_u32(q_s) + i * Sh::kTileBytes + (c >> 3) * (kTile * 128) + r0 * 128 + (((c & 7) ^ (r0 & 7)) << 4);
            RowOf row(row_base + i * kTile + r0, a.G, RS);
            const __half* base = a.q + (long long)seq.row0 * a.q_stride + (long long)kvh * a.G * HD + c * 8;
#pragma unroll 4
            for (int k = 0; k < kTile / RS; ++k, row.step()) {
                const bool ok = i * kTile + r0 + k * RS < rows;
                const __half* src = ok ? base + row.tok * a.q_stride + row.head * HD : a.q;
                cp_async16_zfill(at + k * RS * 128, src, ok ? 16u : 0u);
            }
            cp_async_commit();
            cp_async_wait<0>();
            fence_async_smem();
            mbar_arrive(smem_u32(&bars.q_full[i]));
        }
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + i * kTile + lanes, o_at = tmem + 2 * kTile + i * kTile + lanes;
        const int R = row_base + i * kTile + r;
        const bool valid = i * kTile + r < rows;
        const int tok = R / a.G, head = kvh * a.G + (R - tok * a.G);
        const int limit = valid ? max(0, ctx + tok + 1) : 0;   // this row sees positions [0, limit)
        float m = -INFINITY, l0 = 0.f, l1 = 0.f;
        if (i < n_sub) {
            for (int j = 0; j < n; ++j) {
                tc_wait(&bars.s_full[i], j & 1, &s_abort, fault);
                tc_fence_after();
                uint32_t v[4][32];
#pragma unroll
                for (int h = 0; h < 4; ++h) tmem_ld(s_at + h * 32, v[h]);
                tmem_wait_ld();
#pragma unroll
                for (int h = 0; h < 4; ++h) tmem_pin(v[h]);
                const __half* sc = s_scale[j % Sh::kScales][0];
                if constexpr (Sh::kQuant) {   // K's scales
#pragma unroll
                    for (int h = 0; h < kTile / 8; ++h) {
                        float f[8];
                        scales8(sc + 8 * h, f);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            mul2(v[h >> 2][(8 * h + 2 * e) & 31], v[h >> 2][(8 * h + 2 * e + 1) & 31], f[2 * e], f[2 * e + 1]);
                    }
                }
                const int lim = limit - (t0 + j) * kTile;      // of this tile
                if (__any_sync(0xffffffffu, lim < kTile)) {
#pragma unroll
                    for (int h = 0; h < 4; ++h)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (h * 32 + e >= lim) v[h][e] = __float_as_uint(-INFINITY);
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; ++e)
#pragma unroll
                    for (int h = 0; h < 4; ++h) mx[h] = fmaxf(mx[h], __uint_as_float(v[h][e]));
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                // grow: the old sums are too large a scale off (or there is no scale yet)
                const bool grow = top > m && !((top - m) * a.c <= Sh::kGrow);
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? (m == -INFINITY ? 0.f : ex2((m - top) * a.c)) : 1.f;
                    if (grow) m = top;
                    l0 *= f;
                    l1 *= f;
                    if (j > 0) {   // the products so far are in O: s_full follows them
#pragma unroll
                        for (int h = 0; h < HD / 16; ++h) {
                            uint32_t o[16];
                            tmem_ld(o_at + h * 16, o);
                            tmem_wait_ld();
                            tmem_pin(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st(o_at + h * 16, o);
                        }
                    }
                }
                const float k = m == -INFINITY ? 0.f : -m * a.c;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t w[32];
                    float f[8];
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        float x = __uint_as_float(v[2 * h + (e >> 4)][(2 * e) & 31]);
                        float y = __uint_as_float(v[2 * h + (e >> 4)][(2 * e + 1) & 31]);
                        fma2(x, y, a.c, k);
                        x = ex2(x);
                        y = ex2(y);
                        add2(l0, l1, x, y);
                        if constexpr (Sh::kQuant) {   // V's scales, without their powers of two
                            if (e % 4 == 0) scales8(sc + kTile + h * 64 + 2 * e, f);
                            uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
                            mul2(xb, yb, f[(2 * e) & 7], f[(2 * e + 1) & 7]);
                            w[e] = pack_half2(__uint_as_float(xb), __uint_as_float(yb));
                        } else {
                            w[e] = pack_half2(x, y);
                        }
                    }
                    tmem_st(s_at + h * 32, w);
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(smem_u32(&bars.p_full[i]));
            }
            const float l = l0 + l1;
            if (n > 0) {
                tc_wait(&bars.o_done, 0, &s_abort, fault);
                tc_fence_after();
            }
            const int from = max(all_see, t0 * kTile), to = min(limit, t1 * kTile);   // what this row sees of the masked
            const bool mended = n > 0 && valid && s_mended != 0;
            if (S == 1) {
                const float inv = l > 0.f ? 1.f / l : 0.f;
                // this warp's 32 rows of the output, FP16, in Q's place (every product with Q is done), chunks xor row
                constexpr int CH = HD / 8;
                uint4* stage = reinterpret_cast<uint4*>(q_s) + (size_t)(i * kTile + (warp & 3) * 32) * CH;
#pragma unroll
                for (int h = 0; h < HD / 32; ++h) {
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                    if (n > 0) {
                        tmem_ld(o_at + h * 32, o);
                        tmem_wait_ld();
                        tmem_pin(o);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t w[4];
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            w[x] = pack_half2(__uint_as_float(o[8 * e + 2 * x]) * inv, __uint_as_float(o[8 * e + 2 * x + 1]) * inv);
                        stage[lane * CH + ((h * 4 + e) ^ (lane & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                __syncwarp();
                const int first = row_base + i * kTile + (warp & 3) * 32, c = lane % CH;
                const int count = min(32, rows - (i * kTile + (warp & 3) * 32));
                RowOf row(first + lane / CH, a.G, 32 / CH);
                __half* base = a.out + ((long long)seq.row0 * a.NH + kvh * a.G) * HD + c * 8;
#pragma unroll 4
                for (int x = lane / CH; x < count; x += 32 / CH, row.step())
                    *reinterpret_cast<uint4*>(base + ((long long)row.tok * a.NH + row.head) * HD) = stage[x * CH + (c ^ (x & 7))];
                __syncwarp();
                if (mended) {
                    add_mended<FMT, HD>(p, b, kvh, from, to, a.out + ((long long)(seq.row0 + tok) * a.NH + head) * HD, nullptr,
                                        r, fault);
                }
            } else {
                // this CTA's part of the rows: 16-byte chunks
                // xor the row so that the lanes' stores spread over the banks
                part_m[i * kTile + r] = m;
                part_l[i * kTile + r] = l;
                float4* part = reinterpret_cast<float4*>(part_o) + (size_t)(i * kTile + r) * (HD / 4);
#pragma unroll
                for (int h = 0; h < HD / 32; ++h) {
                    uint32_t o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0u;
                    if (n > 0) {
                        tmem_ld(o_at + h * 32, o);
                        tmem_wait_ld();
                        tmem_pin(o);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        part[(h * 8 + e) ^ (r & (HD / 4 - 1))] =
                            make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                        __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                }
                if (mended) add_mended<FMT, HD>(p, b, kvh, from, to, nullptr, reinterpret_cast<float*>(part), r, fault);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tmem_dealloc(tmem, kTmemCols);
    if (S > 1) {
        cluster.sync();   // every CTA's part is there
        // The softmax warps merge (they hold the registers) this CTA's share of the rows, in rank order: the same bits
        // every time.  First every part's factor per row, then the sums, several loads from the other CTAs in flight.
        const int sub_rows = n_sub * kTile, lo = sub_rows * rank / S, cnt = min(sub_rows * (rank + 1) / S, rows) - lo;
        float* factor = part_l + kItemRows;   // [S][cnt]
        if (warp < kMmaWarp) {
            constexpr int kMerge = kMmaWarp * 32;
            for (int x = threadIdx.x; x < cnt; x += kMerge) {
                float mu[kMaxSplit], lu[kMaxSplit], M = -INFINITY, L = 0.f;
#pragma unroll
                for (int u = 0; u < kMaxSplit; ++u) {
                    mu[u] = u < S ? cluster.map_shared_rank(part_m, u)[lo + x] : -INFINITY;
                    lu[u] = u < S ? cluster.map_shared_rank(part_l, u)[lo + x] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < kMaxSplit; ++u) M = fmaxf(M, mu[u]);
#pragma unroll
                for (int u = 0; u < kMaxSplit; ++u) {
                    mu[u] = mu[u] == -INFINITY ? 0.f : ex2((mu[u] - M) * a.c);   // 0: nothing seen there
                    L = fmaf(lu[u], mu[u], L);
                }
                const float inv = L > 0.f ? 1.f / L : 0.f;
#pragma unroll
                for (int u = 0; u < kMaxSplit; ++u)
                    if (u < S) factor[u * cnt + x] = mu[u] * inv;
            }
            named_bar_sync(2, kMerge);
            constexpr int CH = HD / 4, kBatch = 4;
            for (int x0 = threadIdx.x; x0 < cnt * CH; x0 += kBatch * kMerge) {
                float4 o[kBatch];
#pragma unroll
                for (int y = 0; y < kBatch; ++y) o[y] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                for (int u = 0; u < S; ++u) {
                    const float4* part = reinterpret_cast<const float4*>(cluster.map_shared_rank(part_o, u));
#pragma unroll
                    for (int y = 0; y < kBatch; ++y) {
                        const int x = x0 + y * kMerge, r = x / CH, ch = x % CH;
                        if (x >= cnt * CH) break;
                        const float4 q = part[(size_t)(lo + r) * CH + (ch ^ ((lo + r) & (CH - 1)))];
                        const float f = factor[u * cnt + r];
                        o[y].x = fmaf(q.x, f, o[y].x);
                        o[y].y = fmaf(q.y, f, o[y].y);
                        o[y].z = fmaf(q.z, f, o[y].z);
                        o[y].w = fmaf(q.w, f, o[y].w);
                    }
                }
#pragma unroll
                for (int y = 0; y < kBatch; ++y) {
                    const int x = x0 + y * kMerge, r = x / CH, ch = x % CH;
                    if (x >= cnt * CH) break;
                    const int R = row_base + lo + r, tok = R / a.G;
                    __half* dst =
                        a.out + ((long long)(seq.row0 + tok) * a.NH + kvh * a.G + R - tok * a.G) * HD + ch * 4;
                    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(o[y].x, o[y].y), pack_half2(o[y].z, o[y].w));
                }
            }
        }
        cluster.sync();   // no CTA leaves while another reads its part
    }
}

// cuTensorMapEncodeTiled, taken from the driver at run time (the library does not link against it).
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encode(cudaError_t* err) {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
    auto f = fn.load(std::memory_order_acquire);
    *err = cudaSuccess;
    if (f == nullptr) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult res = cudaDriverEntryPointSymbolNotFound;
        *err = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &ptr, 12000, cudaEnableDefault, &res);
        if (*err == cudaSuccess && (res != cudaDriverEntryPointSuccess || ptr == nullptr)) *err = cudaErrorNotSupported;
        if (*err != cudaSuccess) return nullptr;
        f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
        fn.store(f, std::memory_order_release);
    }
    return f;
}

// The pool's K or V as a tensor [page][kv head][panel][slot][row bytes]: a box is one page's (at most 128) slots of one
// head and one 128-byte panel (FP16) or whole vector (codes).
template <int FMT, int HD>
cudaError_t pool_map(CUtensorMap* map, const uint8_t* base, const Paged& p) {
    cudaError_t e;
    auto encode = tensor_map_encode(&e);
    if (encode == nullptr) return e;
    constexpr bool quant = FMT != AF_KV_F16;
    constexpr int esz = KvFormat<FMT>::kBytes, inner = quant ? HD : 64, panels = HD / inner;
    const cuuint64_t row = (cuuint64_t)p.NKV * HD * esz;
    const int page = 1 << p.page_shift;
    const cuuint64_t dims[5] = {(cuuint64_t)inner, (cuuint64_t)page, (cuuint64_t)panels, (cuuint64_t)p.NKV,
                                (cuuint64_t)std::max(1, p.n_pages)};
    const cuuint64_t strides[4] = {row, (cuuint64_t)inner * esz, (cuuint64_t)HD * esz, (cuuint64_t)p.page_bytes};
    const cuuint32_t box[5] = {(cuuint32_t)inner, (cuuint32_t)std::min(page, kTile), 1, 1, 1};
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    const CUresult r = encode(map, quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                              const_cast<uint8_t*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              quant ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

template <int FMT, int HD>
cudaError_t launch(const Paged& p, const TcArgs& a, unsigned clusters, int S, unsigned* fault, cudaStream_t st) {
    auto kernel = paged_chunk_kernel<FMT, HD>;
    using Sh = Shape<FMT, HD>;
    static std::atomic<bool> set[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !set[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Sh::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxDevices) set[dev].store(true, std::memory_order_release);
    }
    CUtensorMap k_map, v_map;
    e = pool_map<FMT, HD>(&k_map, p.k, p);
    if (e == cudaSuccess) e = pool_map<FMT, HD>(&v_map, p.v, p);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(clusters * S);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = Sh::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p, a, k_map, v_map, fault);
}

}  // namespace

// Launches the chunk kernel over every sequence of more than skip_rows rows.
cudaError_t paged_chunk_launch(int format, int head_dim, const Paged& p, const void* q, long long q_stride, int n_heads,
                               float scale, int skip_rows, int max_kv, void* out, unsigned* fault, cudaStream_t st) {
    TcArgs a{};
    a.q = static_cast<const __half*>(q);
    a.q_stride = q_stride;
    a.out = static_cast<__half*>(out);
    a.NH = n_heads;
    a.G = n_heads / p.NKV;
    a.c = scale * 1.4426950408889634f;
    a.skip_rows = skip_rows;
    const long long rows = (long long)p.n_tokens * a.G;
    // row tile pairs at most: each sequence ends one early, and has more than skip_rows rows
    const long long seqs = std::min<long long>(p.n_seqs, rows / (skip_rows + 1));
    const long long items = rows / kItemRows + seqs;
    const long long clusters = items * p.NKV;
    if (items == 0) return cudaSuccess;
    const long long full_items = std::max((rows + kItemRows - 1) / kItemRows, seqs) * p.NKV;
    const int S = paged_chunk_split(full_items, std::max(1, (max_kv + kTile - 1) / kTile), device_sm_count());
    if (clusters * S > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    auto go = [&](auto fmt) {
        return head_dim == 128 ? launch<decltype(fmt)::value, 128>(p, a, (unsigned)clusters, S, fault, st)
                               : launch<decltype(fmt)::value, 64>(p, a, (unsigned)clusters, S, fault, st);
    };
    if (format == AF_KV_F16) return go(std::integral_constant<int, AF_KV_F16>());
    if (format == AF_KV_FP8_E4M3) return go(std::integral_constant<int, AF_KV_FP8_E4M3>());
    return go(std::integral_constant<int, AF_KV_INT8>());
}

}  // namespace af

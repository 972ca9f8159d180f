// af_paged_few.cu -- attention of few rows per sequence (a decoded token, a few
// drafted ones) over a paged KV cache: af_paged_attention's path for sequences
// of at most 16 (token, query head) rows per kv head.
//
// The floor is reading the cache once (one token over 131,001 FP8 positions, 8 heads of 128:
// 54.5 us in a graph, 58.5 to 59.5 among other calls, 5.0 and 4.6 TB/s; 64 ragged INT8 sequences of up to 8000: 127 us,
// 5.1 TB/s, and 133 to 143).  An item is one (sequence, kv head); its
// positions go in tiles of 16, each of a CTA's W warps taking every W-th tile of
// the CTA's range in a cp.async ring of its own (no CTA-wide barrier in the loop).
// The work is divided over CTAs in one of two ways:
//   * clusters (short caches): S CTAs share an item and merge through distributed
//     shared memory -- one launch, no workspace;
//   * one wave (long caches, with a workspace): all items' tiles in a row, cut
//     into equal pieces, one per CTA that the GPU holds at once, so neither ragged
//     lengths nor a single long sequence leaves SMs idle.  An item's pieces go to
//     the workspace and a second, dependent launch merges them.  (One sequence of
//     131,001 FP8 positions over 8 heads: clusters of 16, of which the GPU holds
//     7, took 102 us.)
// Per tile, on m16n8k16 MMAs with the roles swapped so that 8 rows do
// not waste a 16-row operand:
//   S^T [positions x rows] = K Q^T        K from shared memory, Q in registers
//   O^T [dims x rows]     += V^T P^T      P^T turned round by movmatrix
// Both results hold the same rows per lane, so the running maximum, the sum and
// the rescale need no exchange; the maximum itself is only looked for across
// lanes (and O rescaled) when some score exceeds the last one by a factor 2^8 --
// P stays below 2^8, in FP16's exact range.
//   * 8-bit K goes from 16-byte words to A operands without a transpose: the
//     MMA's k index is a sum, so its order is chosen as the bytes lie (Q is
//     loaded in that order).  8-bit V pairs positions by byte permutes.
//   * INT8 codes are exact FP16 operands: the byte as a mantissa of 1024, less
//     1152.  (Left in the operand and taken out of the accumulator as 1152 sum(q),
//     the offset costs no instruction, but the accumulator then rounds at its
//     size, up to 2^10 times the score's for a query that leans to one side.)
//   * P is rounded to FP16, the second MMA's operand (relative error of the output
//     2.7e-4 to 2.9e-4, where its own rounding alone makes 2.1e-4).
//   * K's scale multiplies S in FP32.  V's is split: its power of two into the
//     codes' FP16 operands, exactly, the rest, in [1, 2), into P before its one
//     rounding.  A position's weight so keeps its 11 bits whatever the scales
//     around it are.  (With all of it in P, brought to about 1 by a power of two
//     of the warp's, one vector of zeros, whose scale is 1, left the others'
//     weights the bits of FP16's subnormals.)
//   * Warps and CTAs merge in a fixed order: the same bits every time.
//   * The loop is bound by the latency of a warp's steps: 8 warps per SM (two per
//     scheduler) issued in 45% of the cycles and read the cache at 3.6 TB/s, so
//     the rings are short and the registers few enough for 16 (12 with 16 rows
//     of 128 dims), which issue in 56 to 58% and keep DRAM 63% busy.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "af_paged.cuh"

namespace af {
namespace {

constexpr int kMaxSplit = 8;
constexpr int kMergeThreads = 512;  // at most
constexpr int KT = 16;             // positions of a tile
constexpr int kLong = 2560;        // positions per CTA of a cluster past which the work is cut into one wave (16 FP16
                                   // sequences of 4096 over 8 heads: clusters of 2 44 us, wave 48; 4 FP8 of 32768:
                                   // clusters of 8 71 us, wave 54; 48 ragged FP16 ones of up to 4099, 4 rows:
                                   // clusters of 2 31 us, wave 33)

// NT: 8-row column tiles; BIG: one CTA per SM with all its warps, else CTAs of four warps.
template <int FMT, int HD, int NT, bool BIG>
struct Few {
    static constexpr int kEsz = KvFormat<FMT>::kBytes;
    static constexpr int kRow = HD * kEsz;            // bytes of a head vector
    static constexpr int kCh = kRow / 16;             // its 16-byte chunks
    static constexpr int kHalf = KT * kRow;           // K (or V) bytes of a stage
    // CTAs of four warps per SM: registers (128 or 168 per thread) and ring bytes follow
    static constexpr int kPerSm = (NT == 2 || FMT == AF_KV_F16) && HD == 128 ? 3 : 4;
    static constexpr int W = BIG ? 4 * kPerSm : 4;
    static constexpr int kThreads = W * 32;
    static constexpr int kMinCtas = BIG ? 1 : kPerSm;
    static constexpr int kRing = kPerSm == 4 ? 12 * 1024 : 16 * 1024;
    static constexpr int kStages = kRing / (2 * kHalf);
    static constexpr size_t kSmem = (size_t)W * kStages * 2 * kHalf;
    // log2 of the growth of a score over the maximum that moves it: P times the rest of any finite scale stays finite
    // in FP16 (2^7 * 511.75, 2^5 * 2047)
    static constexpr float kGrow = FMT == AF_KV_F16 ? 8.f : FMT == AF_KV_FP8_E4M3 ? 7.f : 5.f;
    // Byte offset of chunk ch of row r in a tile.  The chunks of each 128-byte line are permuted so that the lanes
    // of one shared-memory access fall into different banks: FP16 rows are read by ldmatrix (8 rows, one chunk);
    // 8-bit K two rows by four chunks; 8-bit V four even (or odd) rows by 32 bytes.
    __device__ static __forceinline__ uint32_t at(int r, int ch, bool is_v) {
        const int x = r * kCh + ch, line = x >> 3, cc = x & 7;
        const int f = FMT == AF_KV_F16 ? r & 7
                      : HD == 64       ? (line & 3) << 1
                      : is_v           ? ((r >> 1) & 3) << 1
                                       : (r & 1) << 2;
        return (uint32_t)(line * 128 + ((cc ^ f) << 4));
    }
};

struct FewArgs {
    const __half* q;
    long long q_stride;
    __half* out;
    int NH, G;
    float c;       // scale * log2(e)
    int alone;     // no other kernel takes the sequences of too many rows: record them
    int behind;    // launched while another kernel of the call may still run: end after it
    // one wave: partial O [2 ctas][ROWS][HD], m and l [2 ctas][ROWS], and for each CTA the item that begins in it and
    // goes on in the next ones: {first row, kv head, pieces (0: no such item), rows}
    float4* part_o;
    float2* part_ml;
    int4* part_head;
    int ctas;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// E4M3's NaN codes -> 0; whether there were any.
__device__ __forceinline__ bool mend_codes(uint4& v) {
    uint32_t* w = &v.x;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t nan = __vcmpeq4(w[i] & 0x7f7f7f7fu, 0x7f7f7f7fu);
        any |= nan != 0;
        w[i] &= ~nan;
    }
    return any;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t movm(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, uint32_t n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// The largest power of two of V's scale that goes into the codes: for INT8 the byte stands on 1152, whose product with
// the power has to be an FP16 value.
template <int FMT>
constexpr int kPowerMax = FMT == AF_KV_INT8 ? 5 : 7;
// Four codes times a pair of powers of two (even, odd bytes) -> four FP16 values, exactly.  INT8: the fused product takes
// the 1152 off before the one rounding.
template <int FMT>
__device__ __forceinline__ void unpack4_scaled(uint32_t w, uint32_t power, uint32_t& lo, uint32_t& hi) {
    const __half2 p = *reinterpret_cast<const __half2*>(&power);
    if constexpr (FMT == AF_KV_INT8) {
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 off = __hmul2(p, __float2half2_rn(-1152.f));
        const __half2 ra = __hfma2(*reinterpret_cast<const __half2*>(&a), p, off);
        const __half2 rb = __hfma2(*reinterpret_cast<const __half2*>(&b), p, off);
        lo = *reinterpret_cast<const uint32_t*>(&ra);
        hi = *reinterpret_cast<const uint32_t*>(&rb);
    } else {
        kv_unpack4<FMT>(w, lo, hi);
        lo = mul_half2(lo, p);
        hi = mul_half2(hi, p);
    }
}

// ---- one wave: every item's tiles in a row, sequence by sequence, head by head ----
// Tiles of one head of sequence b; 0: not a sequence of ours.  (One without positions has an empty tile: its rows are
// zeros that someone has to write.)
template <int ROWS>
__device__ __forceinline__ int few_tiles(const Paged& p, const FewArgs& a, int b, unsigned* fault) {
    const PagedSeq s = paged_seq(p, b, fault);
    const long long rows = (long long)s.q * a.G;
    if (rows == 0 || rows > ROWS) {
        if (rows > ROWS && a.alone) atomicOr(fault, (unsigned)AF_FAULT_PAGED);
        return 0;
    }
    return max(1, (s.kv + KT - 1) / KT);
}
// A CTA's piece of the wave: tiles [lo, hi) of the row of all, beginning in sequence b (-1: nothing), whose first tile
// is `first`.  The item that begins in the piece and goes on ends `tiles - 1` later, in CTA (its last tile) / share,
// or, where all sequences are as long (`even` > 0), after `even` CTAs: each item is then cut into that many pieces at
// its own borders, so that no CTA has parts of two.
struct FewPiece {
    long long lo, hi, first, share;
    int b, even;
};
// By one whole warp.
template <int ROWS>
__device__ FewPiece few_piece(const Paged& p, const FewArgs& a, int cta, int W, unsigned* fault) {
    const int lane = threadIdx.x & 31;
    const unsigned all = 0xffffffffu;
    long long heads = 0;                 // tiles of one head of every sequence
    int low = INT_MAX, high = 0, t0 = 0; // t0: of sequence `lane`, kept where that is all there is
    for (int b = lane; b < p.n_seqs; b += 32) {
        const int t = few_tiles<ROWS>(p, a, b, fault);
        if (b == lane) t0 = t;
        heads += t;
        low = min(low, t);
        high = max(high, t);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) heads += __shfl_xor_sync(all, heads, x);
    low = __reduce_min_sync(all, low);
    high = __reduce_max_sync(all, high);
    FewPiece r{0, 0, 0, 1, -1, 0};
    const long long total = heads * p.NKV, items = (long long)p.n_seqs * p.NKV;
    if (total == 0) return r;
    if (low == high && items <= a.ctas) {
        const int k = max(1, (int)min((long long)(a.ctas / items), (long long)low / (2 * W)));   // two tiles per warp
        const int item = cta / k, piece = cta - item * k;
        if (item >= items) return r;
        r.even = k;
        r.b = item / p.NKV;
        r.first = (long long)r.b * p.NKV * low;
        r.lo = (long long)item * low + (long long)low * piece / k;
        r.hi = (long long)item * low + (long long)low * (piece + 1) / k;
        return r;
    }
    r.share = max((total + a.ctas - 1) / a.ctas, (long long)2 * W);
    r.lo = cta * r.share;
    r.hi = min(total, r.lo + r.share);
    if (r.lo >= r.hi) return r;
    long long seen = 0;
    for (int b0 = 0; b0 < p.n_seqs; b0 += 32) {
        const long long t =
            (long long)(b0 == 0 ? t0 : b0 + lane < p.n_seqs ? few_tiles<ROWS>(p, a, b0 + lane, fault) : 0) * p.NKV;
        long long inc = t;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const long long y = __shfl_up_sync(all, inc, x);
            if (lane >= x) inc += y;
        }
        const unsigned who = __ballot_sync(all, r.lo >= seen + inc - t && r.lo < seen + inc);
        if (who != 0) {
            const int src = __ffs(who) - 1;
            r.first = seen + __shfl_sync(all, inc - t, src);
            r.b = b0 + src;
            return r;
        }
        seen += __shfl_sync(all, inc, 31);
    }
    return r;
}

template <int FMT, int HD, int NT, bool BIG, bool WAVE>
__global__ void __launch_bounds__(Few<FMT, HD, NT, BIG>::kThreads, Few<FMT, HD, NT, BIG>::kMinCtas)
    paged_few_kernel(const Paged p, const FewArgs a, unsigned* fault) {
    namespace cg = cooperative_groups;
    using F = Few<FMT, HD, NT, BIG>;
    constexpr int W = F::W, ROWS = 8 * NT, MT = HD / 16;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float s_m[W][ROWS], s_l[W][ROWS];
    __shared__ float c_m[ROWS], c_l[ROWS];   // this CTA's, for the cluster
    __shared__ int s_mended[W];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    int S = 1, rank = 0, b, kvh, t0, t1;
    PagedSeq seq;
    long long u0 = 0, u1 = 0, first = 0, share = 1;   // one wave: this CTA's piece
    int even = 0;
    // What follows in the stream waits for this grid alone, so the grid must not end before the kernel it was launched
    // behind: its first CTA waits for that one (the others leave, their places are free for more).
    auto leave = [&] {
        if (a.behind && blockIdx.x == 0) pdl_wait();
    };
    if constexpr (WAVE) {
        pdl_launch_dependents();             // every CTA is resident: the merge may line up behind them
        __shared__ FewPiece s_piece;
        if (warp == 0) {
            const FewPiece x = few_piece<ROWS>(p, a, blockIdx.x, W, fault);
            if (lane == 0) {
                s_piece = x;
                a.part_head[blockIdx.x] = make_int4(0, 0, 0, 0);
            }
        }
        __syncthreads();
        b = s_piece.b;
        u0 = s_piece.lo;
        u1 = s_piece.hi;
        first = s_piece.first;
        share = s_piece.share;
        even = s_piece.even;
        if (b < 0) {
            leave();
            return;
        }
    } else {
        cg::cluster_group cluster = cg::this_cluster();
        S = (int)cluster.num_blocks();
        rank = (int)cluster.block_rank();
        const int cid = blockIdx.x / S;
        b = cid / p.NKV;
        kvh = cid - b * p.NKV;
        seq = paged_seq(p, b, fault);
        const long long rows = (long long)seq.q * a.G;
        if (rows == 0 || rows > ROWS) {      // the whole cluster leaves
            if (rows > ROWS && a.alone && threadIdx.x == 0) atomicOr(fault, (unsigned)AF_FAULT_PAGED);
            leave();
            return;
        }
    }
  for (;;) {   // one wave: every piece of an item that falls into this CTA's tiles
    int tiles;
    if constexpr (WAVE) {
        seq = paged_seq(p, b, fault);
        tiles = max(1, (seq.kv + KT - 1) / KT);
        kvh = (int)((u0 - first) / tiles);
        t0 = (int)(u0 - first - (long long)kvh * tiles);
        t1 = (int)min((long long)tiles, t0 + (u1 - u0));
    } else {
        tiles = (seq.kv + KT - 1) / KT;
        t0 = (int)((long long)tiles * rank / S);
        t1 = (int)((long long)tiles * (rank + 1) / S);
    }
    const int rows = seq.q * a.G;
    const int ctx = seq.kv - seq.q, end = seq.kv;    // the last row sees every position
    const int n = (t1 - t0 - warp + W - 1) / W;      // this warp's tiles: t0 + warp + W * j
    const uint32_t ring = smem_u32(smem) + warp * (F::kStages * 2 * F::kHalf);

    // The pages of tile j's two halves of 8 positions (one page unless pages are of 8); -1: none.
    struct Pages {
        int lo, hi;
    };
    const int* table = p.table + paged_table_at(b, p.table_stride, 0, 0);
    auto page_of = [&](int pos) {
        const int page = __ldg(table + (pos >> p.page_shift));
        if (paged_page_ok(page, p.n_pages)) return page;
        atomicOr(fault, (unsigned)AF_FAULT_PAGED);
        return -1;
    };
    auto find = [&](int j) {
        Pages x{-1, -1};
        const int pos = (t0 + warp + W * j) * KT;
        if (j < n && pos < end) {
            x.lo = page_of(pos);
            x.hi = p.page_shift > 3 ? x.lo : pos + 8 < end ? page_of(pos + 8) : -1;
        }
        return x;
    };
    // Copies tile j into its stage: lane l takes chunk l % kCh of every (32 / kCh)-th row.  The rows of one lane are
    // RPI apart, so their places in the stage differ by constants.
    constexpr int RPI = 32 / F::kCh;                 // rows of one warp-wide copy, at most 8
    constexpr int half = 8 / RPI;                    // copies per half tile
    const int row_of = lane / F::kCh;
    const long long row_bytes = (long long)p.NKV * F::kRow, step = RPI * row_bytes;
    const long long lane_off = (long long)row_of * row_bytes + (lane % F::kCh) * 16 + (long long)kvh * F::kRow;
    const uint8_t *k_lane = p.k + lane_off, *v_lane = p.v + lane_off;
    uint32_t k_to[KT / RPI], v_to[KT / RPI];
#pragma unroll
    for (int i = 0; i < KT / RPI; ++i) {
        k_to[i] = F::at(row_of + i * RPI, lane % F::kCh, false);
        v_to[i] = F::kHalf + F::at(row_of + i * RPI, lane % F::kCh, true);
    }
    auto issue = [&](int j, uint32_t stage, Pages pg) {
        if (j < n) {
            const int pos = (t0 + warp + W * j) * KT;
            const long long lo = paged_at(p, max(pg.lo, 0), pos, 0, F::kRow);
            const long long hi = p.page_shift > 3 ? lo + 8 * row_bytes : paged_at(p, max(pg.hi, 0), pos, 0, F::kRow);
            if ((pg.lo | pg.hi) >= 0 && pos + KT <= end) {
#pragma unroll
                for (int i = 0; i < KT / RPI; ++i) {
                    const long long src = (i < half ? lo : hi) + (i % half) * step;
                    cp_async16(stage + k_to[i], k_lane + src);
                    cp_async16(stage + v_to[i], v_lane + src);
                }
            } else {   // positions past the end, or without a page: zeros
#pragma unroll
                for (int i = 0; i < KT / RPI; ++i) {
                    const bool ok = (i < half ? pg.lo : pg.hi) >= 0 && pos + row_of + i * RPI < end;
                    const long long src = ok ? (i < half ? lo : hi) + (i % half) * step : 0;
                    cp_async16_zfill(stage + k_to[i], ok ? k_lane + src : p.k, ok ? 16u : 0u);
                    cp_async16_zfill(stage + v_to[i], ok ? v_lane + src : p.v, ok ? 16u : 0u);
                }
            }
        }
        cp_async_commit();
    };
    // Scales of tile j: lane l < 16 K's of position l, lane 16 + l V's.
    const __half* sc_lane = (lane < 16 ? p.ks : p.vs) + kvh;
    auto scales = [&](int j, Pages pg) {
        __half x = __float2half_rn(0.f);
        if constexpr (FMT != AF_KV_F16) {
            const int pos = (t0 + warp + W * j) * KT + (lane & 15), page = lane & 8 ? pg.hi : pg.lo;
            if (page >= 0 && pos < end) x = __ldg(sc_lane + paged_scale(p, page, pos, 0));
        }
        return x;
    };

    constexpr int D = F::kStages - 1;   // tiles in flight ahead of the one in use
    Pages next = find(0);
    __half sc_ring[D];                  // scales of tiles j .. j + D - 1
#pragma unroll
    for (int j = 0; j < D; ++j) {
        const Pages pg = next;
        next = find(j + 1);
        issue(j, ring + j * (2 * F::kHalf), pg);
        sc_ring[j] = scales(j, pg);
    }

    // Q as the B operand: row nt * 8 + g; the k order of an 8-bit K's bytes, or ldmatrix's
    uint32_t qf[HD / 16][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g, tok = r / a.G;
        const __half* src = a.q + (long long)(seq.row0 + tok) * a.q_stride + (kvh * a.G + r - tok * a.G) * HD;
#pragma unroll
        for (int s = 0; s < HD / 16; ++s) {
            const int d = FMT == AF_KV_F16 ? 16 * s + 2 * c : 64 * (s >> 2) + 16 * c + 4 * (s & 3);
            constexpr int step = FMT == AF_KV_F16 ? 8 : 2;
            qf[s][nt][0] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + d)) : 0u;
            qf[s][nt][1] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(src + d + step)) : 0u;
        }
    }
    // the lane's rows of S^T and O^T: nt * 8 + 2c + e; each sees positions [0, lim)
    int lim[NT][2];
    float m[NT][2], l[NT][2], o[MT][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * c + e;
            lim[nt][e] = r < rows ? max(0, ctx + r / a.G + 1) : 0;
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
        }
    }
    const int seen_by_all = max(0, ctx + 1);         // positions that no row masks
    // Places of the lane's operands in a stage: for 8-bit, the chunks of one row differ by an xor, rows by constants
    // (F::at's permutation of rows 2c, 2c + 1, 2c + 8, 2c + 9, and of g, g + 8, is one).
    const uint32_t k_at = FMT == AF_KV_F16 ? 0u : F::at(g, c, false);
    const uint32_t v_at = FMT == AF_KV_F16 ? 0u : F::at(2 * c, g >> 2, true) + (uint32_t)((g & 3) * 4);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][nt][e] = 0.f;

    bool mended = false;                             // V had infinities or NaN where some row does not look
    uint32_t stage = ring, to = ring + D * (2 * F::kHalf);
    const uint32_t ring_end = ring + F::kStages * (2 * F::kHalf);
    for (int j = 0; j < n; ++j) {
        // the stage that tile j + D goes into was read in the last iteration
        __syncwarp();
        const Pages pg = next;
        next = find(j + D + 1);
        issue(j + D, to, pg);
        const __half sc_new = scales(j + D, pg), sc = sc_ring[0];
#pragma unroll
        for (int x = 0; x + 1 < D; ++x) sc_ring[x] = sc_ring[x + 1];
        sc_ring[D - 1] = sc_new;
        cp_async_wait<D>();
        __syncwarp();
        const uint32_t ks = stage, vs = ks + F::kHalf;
        to = stage;
        stage += 2 * F::kHalf;
        if (stage == ring_end) stage = ring;
        const int pos0 = (t0 + warp + W * j) * KT;

        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
        if constexpr (FMT == AF_KV_F16) {
#pragma unroll
            for (int t = 0; t < HD / 16; ++t) {
                uint32_t f[4];
                ldsm4(f, ks + F::at(lane & 15, 2 * t + (lane >> 4), false));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816(s[nt], f[0], f[1], f[2], f[3], qf[t][nt][0], qf[t][nt][1]);
            }
        } else {
#pragma unroll
            for (int u = 0; u < HD / 64; ++u) {
                const uint4 x = lds128(ks + (k_at ^ (u * 64)));
                const uint4 y = lds128(ks + (k_at ^ (u * 64)) + 8 * F::kRow);
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint32_t a0, a1, a2, a3;
                    kv_unpack4<FMT>(xw[t], a0, a2);
                    kv_unpack4<FMT>(yw[t], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816(s[nt], a0, a1, a2, a3, qf[4 * u + t][nt][0], qf[4 * u + t][nt][1]);
                }
            }
        }
        // scores in the exponent's base 2; positions a row does not see: -inf
        float k0 = a.c, k1 = a.c, v0 = 0.f, v1 = 0.f;
        bool up = false;
        uint32_t pow0 = 0u, pow1 = 0u;               // V's powers of two at positions 2c, 2c + 1 and 2c + 8, 2c + 9
        if constexpr (FMT != AF_KV_F16) {
            const float x = __half2float(sc);
            const KvScaleParts parts = kv_split_scale<FMT, kPowerMax<FMT>>(x);
            k0 *= __shfl_sync(0xffffffffu, x, g);
            k1 *= __shfl_sync(0xffffffffu, x, g + 8);
            v0 = __shfl_sync(0xffffffffu, parts.rest, 16 + g);
            v1 = __shfl_sync(0xffffffffu, parts.rest, 24 + g);
            const uint32_t mine = __half_as_ushort(parts.power);
            const uint32_t pair = __byte_perm(mine, __shfl_down_sync(0xffffffffu, mine, 1), 0x5410);
            pow0 = __shfl_sync(0xffffffffu, pair, 16 + 2 * c);
            pow1 = __shfl_sync(0xffffffffu, pair, 24 + 2 * c);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[nt][e] *= k0;
                s[nt][2 + e] *= k1;
            }
        const bool tail = pos0 + KT > seen_by_all;
        if (tail) {
            if constexpr (FMT != AF_KV_INT8) {   // V there: zeros for infinities and NaN
                for (int x = max(0, seen_by_all - pos0) * F::kCh + lane; x < min(KT, end - pos0) * F::kCh; x += 32) {
                    const uint32_t at = vs + F::at(x / F::kCh, x % F::kCh, true);
                    uint4 y = lds128(at);
                    if (FMT == AF_KV_F16 ? mend_chunk(y) : mend_codes(y)) {
                        mended = true;
                        sts128(at, y);
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (pos0 + g >= lim[nt][e]) s[nt][e] = -INFINITY;
                    if (pos0 + g + 8 >= lim[nt][e]) s[nt][2 + e] = -INFINITY;
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {   // (m = -inf: any score is above it, -inf is not)
                const float t = fmaxf(s[nt][e], s[nt][2 + e]);
                up |= t > m[nt][e] + F::kGrow;
            }
        if (__any_sync(0xffffffffu, up)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float t = fmaxf(m[nt][e], fmaxf(s[nt][e], s[nt][2 + e]));
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
                    const float f = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - t);
                    m[nt][e] = t;
                    l[nt][e] *= f;
#pragma unroll
                    for (int x = 0; x < MT; ++x) {
                        o[x][nt][e] *= f;
                        o[x][nt][2 + e] *= f;
                    }
                }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float base = m[nt][e] == -INFINITY ? 0.f : m[nt][e];   // nothing seen yet: weights exp2(-inf) = 0
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float w = ex2(s[nt][2 * h + e] - base);
                    l[nt][e] += w;
                    s[nt][2 * h + e] = FMT == AF_KV_F16 ? w : w * (h ? v1 : v0);
                }
            }
        if (FMT != AF_KV_F16 && tail) {   // a scale may be an infinity or NaN
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if (pos0 + g >= lim[nt][e]) s[nt][e] = 0.f;
                    if (pos0 + g + 8 >= lim[nt][e]) s[nt][2 + e] = 0.f;
                }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            pb[nt][0] = movm(pack_half2(s[nt][0], s[nt][1]));
            pb[nt][1] = movm(pack_half2(s[nt][2], s[nt][3]));
        }
        if constexpr (FMT == AF_KV_F16) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                uint32_t v[4];
                ldsm4_t(v, vs + F::at((lane & 7) + ((lane >> 4) << 3), 2 * t + ((lane >> 3) & 1), true));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816(o[t][nt], v[0], v[1], v[2], v[3], pb[nt][0], pb[nt][1]);
            }
        } else {
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {   // the lane's dims: 32 d + 4 g + 0..3
                const uint32_t at = vs + (v_at ^ (d * 32));
                const uint32_t w0 = lds32(at), w1 = lds32((HD == 64 ? vs + (v_at ^ (d * 32) ^ 64) : at + F::kRow));
                const uint32_t w8 = lds32(at + 8 * F::kRow);
                const uint32_t w9 = lds32((HD == 64 ? vs + (v_at ^ (d * 32) ^ 64) : at + F::kRow) + 8 * F::kRow);
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // dims 2h and 2h + 1 of the four
                    uint32_t a0, a1, a2, a3;
                    unpack4_scaled<FMT>(__byte_perm(w0, w1, h ? 0x7362 : 0x5140), pow0, a0, a1);
                    unpack4_scaled<FMT>(__byte_perm(w8, w9, h ? 0x7362 : 0x5140), pow1, a2, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * d + h][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                }
            }
        }
    }
    cp_async_wait<0>();
    if constexpr (FMT != AF_KV_INT8) {
        const int any = __any_sync(0xffffffffu, mended);
        if (lane == 0) s_mended[warp] = any;
    }
    __syncthreads();   // every ring is idle: the warps' parts go there, FP32 [warp][row][HD]
    float* part = reinterpret_cast<float*>(smem);
    static_assert((size_t)(W + 1) * ROWS * HD * 4 <= F::kSmem, "parts fit");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = nt * 8 + 2 * c + e;
            float t = l[nt][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t += __shfl_xor_sync(0xffffffffu, t, x);
            if (g == 0) {
                s_m[warp][row] = m[nt][e];
                s_l[warp][row] = t;
            }
#pragma unroll
            for (int t2 = 0; t2 < MT; ++t2)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = FMT == AF_KV_F16 ? 16 * t2 + g + 8 * h : 32 * (t2 >> 1) + 4 * g + 2 * (t2 & 1) + h;
                    part[(warp * ROWS + row) * HD + d] = o[t2][nt][2 * h + e];
                }
        }
    __syncthreads();
    // the warps' parts -> this CTA's (or, alone, the output)
    float4* mine = reinterpret_cast<float4*>(part + W * ROWS * HD);
    auto store = [&](int r, int ch, float4 v, float inv) {
        const int tok = r / a.G;
        __half* dst = a.out + ((long long)(seq.row0 + tok) * a.NH + kvh * a.G + r - tok * a.G) * HD + ch * 4;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
    };
    auto add = [](float4& acc, const float4 v, float f) {
        acc.x = fmaf(v.x, f, acc.x);
        acc.y = fmaf(v.y, f, acc.y);
        acc.z = fmaf(v.z, f, acc.z);
        acc.w = fmaf(v.w, f, acc.w);
    };
    for (int x = threadIdx.x; x < rows * (HD / 4); x += F::kThreads) {
        const int r = x / (HD / 4), ch = x % (HD / 4);
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) M = fmaxf(M, s_m[w][r]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = s_m[w][r] == -INFINITY ? 0.f : ex2(s_m[w][r] - M);
            L = fmaf(s_l[w][r], f, L);
            add(v, reinterpret_cast<const float4*>(part)[(w * ROWS + r) * (HD / 4) + ch], f);
        }
        if constexpr (FMT != AF_KV_INT8) {   // what was taken out of V, for the rows that see it
            int any = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) any |= s_mended[w];
            const int to = any ? min(max(0, ctx + r / a.G + 1), t1 * KT) : 0;
#pragma unroll 1
            for (int pos = max(seen_by_all, t0 * KT); pos < to; ++pos) {
                auto bad = [&](int e) {
                    const float y = v_value<FMT, HD>(p, b, pos, kvh, ch * 4 + e, fault);
                    return fabsf(y) < INFINITY ? 0.f : y;
                };
                v.x += bad(0);
                v.y += bad(1);
                v.z += bad(2);
                v.w += bad(3);
            }
        }
        if (WAVE && t1 - t0 < tiles) {   // a piece of an item: the one that begins it, or a later one
            const long long at = ((long long)2 * blockIdx.x + (t0 == 0 ? 1 : 0)) * ROWS + r;
            a.part_o[at * (HD / 4) + ch] = v;
            if (ch == 0) a.part_ml[at] = make_float2(M, L);
        } else if (S == 1) {
            store(r, ch, v, L > 0.f ? 1.f / L : 0.f);
        } else {
            mine[r * (HD / 4) + ch] = v;
            if (ch == 0) {
                c_m[r] = M;
                c_l[r] = L;
            }
        }
    }
    if constexpr (WAVE) {
        if (t0 == 0 && t1 < tiles && threadIdx.x == 0)
            a.part_head[blockIdx.x] =
                make_int4(seq.row0, kvh, even > 0 ? even : (int)((u0 + tiles - 1) / share) - (int)blockIdx.x + 1, rows);
        u0 += t1 - t0;
        if (u0 >= u1) {
            leave();
            return;
        }
        if (u0 - first >= (long long)tiles * p.NKV) {   // on to the next sequence that is ours
            first += (long long)tiles * p.NKV;
            do ++b;
            while (b < p.n_seqs && few_tiles<ROWS>(p, a, b, fault) == 0);
            if (b >= p.n_seqs) {
                leave();
                return;
            }
        }
        __syncthreads();   // the parts have been read: the rings are free
    } else {
        if (S > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();   // every CTA's part is there
            const int total = rows * (HD / 4), lo = total * rank / S, hi = total * (rank + 1) / S;
            for (int x = lo + threadIdx.x; x < hi; x += F::kThreads) {
                const int r = x / (HD / 4), ch = x % (HD / 4);
                float M = -INFINITY, L = 0.f;
                for (int u = 0; u < S; ++u) M = fmaxf(M, cluster.map_shared_rank(c_m, u)[r]);
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
                for (int u = 0; u < S; ++u) {   // rank order: the same bits every time
                    const float mu = cluster.map_shared_rank(c_m, u)[r];
                    const float f = mu == -INFINITY ? 0.f : ex2(mu - M);
                    L = fmaf(cluster.map_shared_rank(c_l, u)[r], f, L);
                    add(v, cluster.map_shared_rank(mine, u)[r * (HD / 4) + ch], f);
                }
                store(r, ch, v, L > 0.f ? 1.f / L : 0.f);
            }
            cluster.sync();   // no CTA leaves while another reads its part
        }
        leave();
        return;
    }
  }
}

// Merges the pieces of the item that begins in CTA blockIdx.x of the wave and goes on in the next ones.  The threads
// divide the outputs and, where those are few, the pieces.
template <int HD, int NT>
__global__ void __launch_bounds__(kMergeThreads) paged_few_merge_kernel(const FewArgs a) {
    constexpr int ROWS = 8 * NT, CH = HD / 4;
    __shared__ float4 s_o[kMergeThreads];
    __shared__ float2 s_ml[kMergeThreads];
    pdl_wait();
    const int4 head = __ldcg(a.part_head + blockIdx.x);
    if (head.z == 0) return;
    const int kvh = head.y, c0 = blockIdx.x, c1 = c0 + head.z - 1;
    const int outs = head.w * CH, groups = max(1, (int)blockDim.x / outs);
    for (int base = 0; base < outs; base += blockDim.x) {
        const int x = base + threadIdx.x % outs, grp = threadIdx.x / outs;
        const bool on = grp < groups && x < outs;
        float M = -INFINITY, L = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        const int r = x / CH, ch = x % CH;
        if (on) {
#pragma unroll 4
            for (int u = c0 + grp; u <= c1; u += groups) {
                const long long at = ((long long)2 * u + (u == c0 ? 1 : 0)) * ROWS + r;
                const float2 ml = __ldcg(a.part_ml + at);
                const float4 y = __ldcg(a.part_o + at * CH + ch);
                const float t = fmaxf(M, ml.x), base_m = t == -INFINITY ? 0.f : t;
                const float f = ex2(M - base_m), h = ex2(ml.x - base_m);
                M = t;
                L = L * f + ml.y * h;
                v.x = v.x * f + y.x * h;
                v.y = v.y * f + y.y * h;
                v.z = v.z * f + y.z * h;
                v.w = v.w * f + y.w * h;
            }
        }
        s_o[threadIdx.x] = v;
        s_ml[threadIdx.x] = make_float2(M, L);
        __syncthreads();
        if (on && grp == 0) {
            float top = -INFINITY;
            for (int u = 0; u < groups; ++u) top = fmaxf(top, s_ml[u * outs + threadIdx.x].x);
            L = 0.f;
            v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int u = 0; u < groups; ++u) {
                const float2 ml = s_ml[u * outs + threadIdx.x];
                const float4 y = s_o[u * outs + threadIdx.x];
                const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
                L = fmaf(ml.y, f, L);
                v.x = fmaf(y.x, f, v.x);
                v.y = fmaf(y.y, f, v.y);
                v.z = fmaf(y.z, f, v.z);
                v.w = fmaf(y.w, f, v.w);
            }
            const float inv = L > 0.f ? 1.f / L : 0.f;
            const int tok = r / a.G;
            __half* dst = a.out + ((long long)(head.x + tok) * a.NH + kvh * a.G + r - tok * a.G) * HD + ch * 4;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_half2(v.x * inv, v.y * inv), pack_half2(v.z * inv, v.w * inv));
        }
        __syncthreads();
    }
}

// How a call's work is divided.
struct FewPlan {
    bool wave, big;
    int S, ctas;
    size_t bytes;   // of workspace (wave)
};
template <int FMT, int HD, int NT>
FewPlan plan(const Paged& p, int max_kv, bool workspace) {
    using F = Few<FMT, HD, NT, false>;
    FewPlan x{};
    const long long items = (long long)p.n_seqs * p.NKV;
    const int sms = std::max(1, device_sm_count());
    const long long slots = (long long)sms * F::kPerSm;
    // Clusters: one wave of CTAs, each with 64 positions at least (2 FP8 sequences of 4096 over 8 heads: 1 / 2 / 4 / 8
    // CTAs per item 47 / 27 / 16 / 12 us; 16 of 8192: 117 / 70 / 54 us, and 59 at 8, past one wave).
    x.S = 1;
    while (x.S < kMaxSplit && items * x.S * 2 <= slots && max_kv >= x.S * 2 * 64) x.S *= 2;
    // One wave, where a CTA of a cluster would have more than kLong positions; big CTAs (one per SM, fewer pieces to
    // merge) where each item is cut into four at least.
    x.wave = workspace && (long long)max_kv > (long long)x.S * kLong;
    x.big = x.wave && items * 4 <= sms;
    x.ctas = (int)(x.big ? sms : slots);   // as many as the GPU holds
    x.bytes = x.wave ? (size_t)x.ctas * (2 * 8 * NT * (HD * 4 + 8) + 16) : 0;
    return x;
}

template <int FMT, int HD, int NT, bool BIG, bool WAVE>
cudaError_t launch_as(const Paged& p, const FewArgs& a, const FewPlan& x, unsigned* fault, cudaStream_t st) {
    using F = Few<FMT, HD, NT, BIG>;
    auto kernel = paged_few_kernel<FMT, HD, NT, BIG, WAVE>;
    static std::atomic<bool> set[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !set[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::kSmem);
        if (e != cudaSuccess) return e;
        if (dev < kMaxDevices) set[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = WAVE ? dim3(x.ctas) : dim3((unsigned)p.n_seqs * p.NKV * x.S);
    cfg.blockDim = dim3(F::kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (!WAVE) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = x.S;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (a.behind) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    e = cudaLaunchKernelEx(&cfg, kernel, p, a, fault);
    if (e != cudaSuccess || !WAVE) return e;
    return launch_pdl(paged_few_merge_kernel<HD, NT>, dim3(x.ctas), dim3(BIG ? kMergeThreads : 256), 0, st, a);
}

template <int FMT, int HD, int NT>
cudaError_t launch(const Paged& p, FewArgs a, int max_kv, void* workspace, size_t bytes, unsigned* fault, cudaStream_t st) {
    if ((long long)p.n_seqs * p.NKV * kMaxSplit > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    FewPlan x = plan<FMT, HD, NT>(p, max_kv, true);
    if (x.wave && (workspace == nullptr || bytes < x.bytes)) x = plan<FMT, HD, NT>(p, max_kv, false);
    if (!x.wave) return launch_as<FMT, HD, NT, false, false>(p, a, x, fault, st);
    a.ctas = x.ctas;
    a.part_o = static_cast<float4*>(workspace);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + (size_t)2 * x.ctas * 8 * NT * (HD / 4));
    a.part_head = reinterpret_cast<int4*>(a.part_ml + (size_t)2 * x.ctas * 8 * NT);
    return x.big ? launch_as<FMT, HD, NT, true, true>(p, a, x, fault, st)
                 : launch_as<FMT, HD, NT, false, true>(p, a, x, fault, st);
}

// Calls f<FMT, HD, NT>() for a call's format, head size and rows.
template <class F>
auto dispatch(int format, int head_dim, int rows_bound, F&& f) {
    auto nt = [&](auto fmt, auto hd) {
        return rows_bound <= 8 ? f(fmt, hd, std::integral_constant<int, 1>()) : f(fmt, hd, std::integral_constant<int, 2>());
    };
    auto hd = [&](auto fmt) {
        return head_dim == 128 ? nt(fmt, std::integral_constant<int, 128>()) : nt(fmt, std::integral_constant<int, 64>());
    };
    if (format == AF_KV_F16) return hd(std::integral_constant<int, AF_KV_F16>());
    if (format == AF_KV_FP8_E4M3) return hd(std::integral_constant<int, AF_KV_FP8_E4M3>());
    return hd(std::integral_constant<int, AF_KV_INT8>());
}

}  // namespace

size_t paged_few_workspace(int format, int head_dim, const Paged& p, int rows_bound, int max_kv) {
    return dispatch(format, head_dim, rows_bound, [&](auto fmt, auto hd, auto nt) {
        return plan<decltype(fmt)::value, decltype(hd)::value, decltype(nt)::value>(p, max_kv, true).bytes;
    });
}

cudaError_t paged_few_launch(int format, int head_dim, const Paged& p, const void* q, long long q_stride, int n_heads,
                             float scale, int rows_bound, bool behind, int max_kv, void* out, void* workspace,
                             size_t workspace_bytes, unsigned* fault, cudaStream_t st) {
    FewArgs a{};
    a.q = static_cast<const __half*>(q);
    a.q_stride = q_stride;
    a.out = static_cast<__half*>(out);
    a.NH = n_heads;
    a.G = n_heads / p.NKV;
    a.c = scale * 1.4426950408889634f;
    a.alone = behind ? 0 : 1;
    a.behind = behind ? 1 : 0;
    return dispatch(format, head_dim, rows_bound, [&](auto fmt, auto hd, auto nt) {
        return launch<decltype(fmt)::value, decltype(hd)::value, decltype(nt)::value>(p, a, max_kv, workspace,
                                                                                      workspace_bytes, fault, st);
    });
}

}  // namespace af

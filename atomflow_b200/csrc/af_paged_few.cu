// af_paged_few.cu -- attention of few rows per sequence (a decoded token, a few
// drafted ones) over a paged KV cache: af_paged_attention's path for sequences
// of at most 16 (token, query head) rows per kv head.
//
// Bound by reading the cache once.  A cluster of S CTAs takes one (sequence, kv
// head); each CTA a contiguous share of its positions, each of its warps every
// W-th tile of 16 positions, in a cp.async ring of its own (no CTA-wide barrier in
// the loop).  Per tile, on m16n8k16 MMAs with the roles swapped so that 8 rows do
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
//   * INT8 K is used as 1024 + code + 128, the byte as an FP16 mantissa; the
//     accumulator starts at -1152 sum(q), which takes the offset out again.
//   * K's scale multiplies S in FP32; V is scaled into FP16 (the values
//     af_paged_kv_read returns), as P has no room for a scale that may be
//     subnormal in FP16.  P is rounded to FP16.
//   * Warps merge in shared memory, CTAs through distributed shared memory, in
//     order: one launch, no workspace, the same bits every time.
//   * The loop is bound by issue slots as much as by DRAM: 8 warps per SM (two per
//     scheduler) issued in 45% of the cycles and read the cache at 3.6 TB/s, so
//     the rings are short and the registers few enough for 16 (12 with 16 rows
//     of 128 dims).
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "af_paged.cuh"

namespace af {
namespace {

constexpr int kMaxSplit = 16;
constexpr int KT = 16;             // positions of a tile
constexpr float kGrow = 8.f;       // log2 of the growth of a score over the maximum that moves it

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

// Four INT8 codes -> 1152 + code as FP16 (two words).
__device__ __forceinline__ void unpack4_offset(uint32_t w, uint32_t& lo, uint32_t& hi) {
    w ^= 0x80808080u;
    lo = __byte_perm(w, 0x64646464u, 0x4140);
    hi = __byte_perm(w, 0x64646464u, 0x4342);
}

template <int FMT, int HD, int NT, bool BIG>
__global__ void __launch_bounds__(Few<FMT, HD, NT, BIG>::kThreads, Few<FMT, HD, NT, BIG>::kMinCtas)
    paged_few_kernel(const Paged p, const FewArgs a, unsigned* fault) {
    namespace cg = cooperative_groups;
    using F = Few<FMT, HD, NT, BIG>;
    constexpr int W = F::W, ROWS = 8 * NT, MT = HD / 16;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float s_m[W][ROWS], s_l[W][ROWS];
    __shared__ float c_m[ROWS], c_l[ROWS];   // this CTA's, for the cluster
    cg::cluster_group cluster = cg::this_cluster();
    const int S = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int cid = blockIdx.x / S, b = cid / p.NKV, kvh = cid - b * p.NKV;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    const PagedSeq seq = paged_seq(p, b, fault);
    const int rows = (int)min((long long)seq.q * a.G, (long long)ROWS + 1);
    if (rows == 0 || rows > ROWS) {   // the whole cluster leaves
        if (rows > ROWS && a.alone && threadIdx.x == 0) atomicOr(fault, (unsigned)AF_FAULT_PAGED);
        return;
    }
    const int ctx = seq.kv - seq.q, end = seq.kv;    // the last row sees every position
    const int tiles = (end + KT - 1) / KT;
    const int t0 = (int)((long long)tiles * rank / S), t1 = (int)((long long)tiles * (rank + 1) / S);
    const int n = (t1 - t0 - warp + W - 1) / W;      // this warp's tiles: t0 + warp + W * j
    const uint32_t ring = smem_u32(smem) + warp * (F::kStages * 2 * F::kHalf);

    // The pages of tile j's two halves of 8 positions (one page unless pages are of 8); -1: none.
    struct Pages {
        int lo, hi;
    };
    auto find = [&](int j) {
        Pages x{-1, -1};
        const int pos = (t0 + warp + W * j) * KT;
        if (j < n) {
            x.lo = paged_page(p, b, pos, fault);
            x.hi = p.page_shift > 3 ? x.lo : pos + 8 < end ? paged_page(p, b, pos + 8, fault) : -1;
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
    auto issue = [&](int j, Pages pg) {
        if (j < n) {
            const int pos = (t0 + warp + W * j) * KT;
            const uint32_t stage = ring + (j % F::kStages) * (2 * F::kHalf);
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
    auto scales = [&](int j, Pages pg) {
        __half x = __float2half_rn(0.f);
        if constexpr (FMT != AF_KV_F16) {
            const int pos = (t0 + warp + W * j) * KT + (lane & 15), page = lane & 8 ? pg.hi : pg.lo;
            if (page >= 0 && pos < end) x = __ldg((lane < 16 ? p.ks : p.vs) + paged_scale(p, page, pos, kvh));
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
        issue(j, pg);
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
    float m[NT][2], l[NT][2], s0[NT][2], o[MT][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        float sum = 0.f;
        if constexpr (FMT == AF_KV_INT8) {   // sum(q) of row nt * 8 + g, then of the lane's rows
#pragma unroll
            for (int s = 0; s < HD / 16; ++s)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&qf[s][nt][e]));
                    sum += x.x + x.y;
                }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * c + e;
            lim[nt][e] = r < rows ? max(0, ctx + r / a.G + 1) : 0;
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
            s0[nt][e] = FMT == AF_KV_INT8 ? -1152.f * __shfl_sync(0xffffffffu, sum, (2 * c + e) * 4) : 0.f;
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

    for (int j = 0; j < n; ++j) {
        // the stage that tile j + D goes into was read in the last iteration
        __syncwarp();
        const Pages pg = next;
        next = find(j + D + 1);
        issue(j + D, pg);
        const __half sc_new = scales(j + D, pg), sc = sc_ring[0];
#pragma unroll
        for (int x = 0; x + 1 < D; ++x) sc_ring[x] = sc_ring[x + 1];
        sc_ring[D - 1] = sc_new;
        cp_async_wait<D>();
        __syncwarp();
        const uint32_t ks = ring + (j % F::kStages) * (2 * F::kHalf), vs = ks + F::kHalf;
        const int pos0 = (t0 + warp + W * j) * KT;

        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = s0[nt][e & 1];
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
                    if constexpr (FMT == AF_KV_INT8) {
                        unpack4_offset(xw[t], a0, a2);
                        unpack4_offset(yw[t], a1, a3);
                    } else {
                        kv_unpack4<FMT>(xw[t], a0, a2);
                        kv_unpack4<FMT>(yw[t], a1, a3);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816(s[nt], a0, a1, a2, a3, qf[4 * u + t][nt][0], qf[4 * u + t][nt][1]);
                }
            }
        }
        // scores in the exponent's base 2; positions a row does not see: -inf
        float k0 = a.c, k1 = a.c;
        if constexpr (FMT != AF_KV_F16) {
            k0 *= __half2float(__shfl_sync(0xffffffffu, sc, g));
            k1 *= __half2float(__shfl_sync(0xffffffffu, sc, g + 8));
        }
        bool up = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[nt][e] *= k0;
                s[nt][2 + e] *= k1;
            }
        if (pos0 + KT > seen_by_all) {
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
                up |= t > m[nt][e] + kGrow;
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
                    s[nt][2 * h + e] = w;
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
            const int k = 2 * c;
            const __half2 s01 = __halves2half2(__shfl_sync(0xffffffffu, sc, 16 + k), __shfl_sync(0xffffffffu, sc, 17 + k));
            const __half2 s89 = __halves2half2(__shfl_sync(0xffffffffu, sc, 24 + k), __shfl_sync(0xffffffffu, sc, 25 + k));
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {   // the lane's dims: 32 d + 4 g + 0..3
                const uint32_t at = vs + (v_at ^ (d * 32));
                const uint32_t w0 = lds32(at), w1 = lds32((HD == 64 ? vs + (v_at ^ (d * 32) ^ 64) : at + F::kRow));
                const uint32_t w8 = lds32(at + 8 * F::kRow);
                const uint32_t w9 = lds32((HD == 64 ? vs + (v_at ^ (d * 32) ^ 64) : at + F::kRow) + 8 * F::kRow);
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // dims 2h and 2h + 1 of the four
                    uint32_t a0, a1, a2, a3;
                    kv_unpack4<FMT>(__byte_perm(w0, w1, h ? 0x7362 : 0x5140), a0, a1);
                    kv_unpack4<FMT>(__byte_perm(w8, w9, h ? 0x7362 : 0x5140), a2, a3);
                    a0 = mul_half2(a0, s01);
                    a1 = mul_half2(a1, s01);
                    a2 = mul_half2(a2, s89);
                    a3 = mul_half2(a3, s89);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816(o[2 * d + h][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
                }
            }
        }
    }
    cp_async_wait<0>();
    __syncthreads();   // every ring is idle: the warps' parts go there, FP32 [warp][row][HD]
    float* part = reinterpret_cast<float*>(smem);
    static_assert((size_t)(W + 1) * ROWS * HD * 4 <= F::kSmem, "parts fit");
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int r = nt * 8 + 2 * c + e;
            float t = l[nt][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) t += __shfl_xor_sync(0xffffffffu, t, x);
            if (g == 0) {
                s_m[warp][r] = m[nt][e];
                s_l[warp][r] = t;
            }
#pragma unroll
            for (int t2 = 0; t2 < MT; ++t2)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = FMT == AF_KV_F16 ? 16 * t2 + g + 8 * h : 32 * (t2 >> 1) + 4 * g + 2 * (t2 & 1) + h;
                    part[(warp * ROWS + r) * HD + d] = o[t2][nt][2 * h + e];
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
        if (S == 1) {
            store(r, ch, v, L > 0.f ? 1.f / L : 0.f);
        } else {
            mine[r * (HD / 4) + ch] = v;
            if (ch == 0) {
                c_m[r] = M;
                c_l[r] = L;
            }
        }
    }
    if (S > 1) {
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
}

template <int FMT, int HD, int NT, bool BIG>
cudaError_t launch_as(const Paged& p, const FewArgs& a, int S, unsigned* fault, cudaStream_t st) {
    using F = Few<FMT, HD, NT, BIG>;
    auto kernel = paged_few_kernel<FMT, HD, NT, BIG>;
    static std::atomic<bool> set[kMaxDevices];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev >= kMaxDevices || !set[dev].load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F::kSmem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        if (dev < kMaxDevices) set[dev].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)p.n_seqs * p.NKV * S);
    cfg.blockDim = dim3(F::kThreads);
    cfg.dynamicSmemBytes = F::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = S;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p, a, fault);
}

template <int FMT, int HD, int NT>
cudaError_t launch(const Paged& p, const FewArgs& a, int max_kv, unsigned* fault, cudaStream_t st) {
    const long long items = (long long)p.n_seqs * p.NKV;
    const int sms = device_sm_count();
    constexpr int W = Few<FMT, HD, NT, true>::W;
    if (items * kMaxSplit > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    // Few items over long caches: even 16 CTAs of four warps each leave most of an SM's warps out, so one big CTA
    // per SM (each warp keeps at least four tiles).
    if (items * kMaxSplit * 4 < (long long)sms * W && max_kv >= kMaxSplit * W * KT * 4)
        return launch_as<FMT, HD, NT, true>(p, a, kMaxSplit, fault, st);
    // Else split until the GPU has several waves of CTAs (sequences differ in length), each warp keeping a tile.
    const long long slots = (long long)sms * Few<FMT, HD, NT, false>::kPerSm;
    int S = 1;
    while (S < kMaxSplit && items * S < 2 * slots && max_kv >= S * 2 * 4 * KT) S *= 2;
    return launch_as<FMT, HD, NT, false>(p, a, S, fault, st);
}

}  // namespace

cudaError_t paged_few_launch(int format, int head_dim, const Paged& p, const void* q, long long q_stride, int n_heads,
                             float scale, int rows_bound, bool alone, int max_kv, void* out, unsigned* fault,
                             cudaStream_t st) {
    FewArgs a{};
    a.q = static_cast<const __half*>(q);
    a.q_stride = q_stride;
    a.out = static_cast<__half*>(out);
    a.NH = n_heads;
    a.G = n_heads / p.NKV;
    a.c = scale * 1.4426950408889634f;
    a.alone = alone ? 1 : 0;
    auto go = [&](auto fmt, auto hd) {
        constexpr int f = decltype(fmt)::value, h = decltype(hd)::value;
        return rows_bound <= 8 ? launch<f, h, 1>(p, a, max_kv, fault, st) : launch<f, h, 2>(p, a, max_kv, fault, st);
    };
    auto hd = [&](auto fmt) {
        return head_dim == 128 ? go(fmt, std::integral_constant<int, 128>()) : go(fmt, std::integral_constant<int, 64>());
    };
    if (format == AF_KV_F16) return hd(std::integral_constant<int, AF_KV_F16>());
    if (format == AF_KV_FP8_E4M3) return hd(std::integral_constant<int, AF_KV_FP8_E4M3>());
    return hd(std::integral_constant<int, AF_KV_INT8>());
}

}  // namespace af

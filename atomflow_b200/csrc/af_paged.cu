// af_paged.cu -- a KV cache in pages for a batch of sequences: rotate, quantise
// and store new tokens (af_paged_kv_write), read positions back
// (af_paged_kv_read), attend over the pages (af_paged_attention).
//
// The batched, paged counterparts of af_rope_kv_write and af_decode_attention:
// one page is a stretch of the same token-major rows [NKV * HD] that the
// one-sequence cache has, so a contiguous cache is a pool whose table counts up.
#include <algorithm>
#include <atomic>
#include <climits>
#include <type_traits>

#include "af_paged.cuh"

using namespace af;

// Fault bits (AF_FAULT_*) of this device's paged kernels, read by af_device_faults.
__device__ unsigned int g_paged_faults;

namespace {

// ---------------------------------------------------------------- write
// A CTA takes a few tokens.  HD / 16 lanes hold one head's vector, lane l the pairs (8l + i, 8l + i + HD/2): RoPE's
// partner is in the same thread, and each load and store of the lanes is one contiguous run.  Bound by DRAM: the qkv
// rows in, q and the codes out.  A token's place is a chain of dependent loads (offsets, length, page): all of a CTA's
// tokens look theirs up at once, one thread each, while the first vectors are on their way, and the vectors of the next
// batch are loaded before those of this one are worked on.  (5 x up to 2047 tokens of 48 heads of 128, FP8, 189 MB:
// 39.5 us, 4.8 TB/s; with one token per CTA 46, with 256 threads 42, with 8-byte loads 41.)
constexpr int kWriteThreads = 128;
constexpr int kWriteBatch = 2;    // vectors of one thread in flight: 32 per CTA at HD 128
constexpr int kWriteTokens = 4;   // tokens of a CTA at most

struct WriteArgs {
    const __half* qkv;
    long long stride;        // elements from one token's row to the next
    const float *cos, *sin;  // [max_seq][HD / 2], or NULL: no rotation
    __half* q_out;
    int NH, max_seq;
    int tokens;              // of a CTA
};

// The framework's rotation (rope.cu of the reference, its fast-math contraction):
// the same two roundings as af_rope_kv_write.
__device__ __forceinline__ void rope_pair(float x, float y, float c, float s, float& o0, float& o1) {
    o0 = fmaf(x, c, -__fmul_rn(y, s));
    o1 = fmaf(x, s, __fmul_rn(y, c));
}

template <int FMT, int HD>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const Paged p, const WriteArgs a,
                                                                    unsigned* fault) {
    constexpr int L = HD / 16, GROUPS = kWriteThreads / L, HALF = HD / 2;
    __shared__ int s_pos[kWriteTokens], s_page[kWriteTokens];   // page -1: nothing to do
    const int t0 = blockIdx.x * a.tokens, nt = min(a.tokens, p.n_tokens - t0);
    const int grp = threadIdx.x / L, l = threadIdx.x % L;
    const bool rotate = a.cos != nullptr;
    const int first = rotate ? 0 : a.NH, nvec = a.NH + 2 * p.NKV;   // without rotation q stays where it is
    struct Batch {
        uint4 lo[kWriteBatch], hi[kWriteBatch];
    };
    auto load = [&](Batch& x, int t, int v0) {
        const __half* row = a.qkv + (long long)(t0 + t) * a.stride + 8 * l;
#pragma unroll
        for (int i = 0; i < kWriteBatch; ++i) {
            const int v = v0 + i * GROUPS;
            x.lo[i] = x.hi[i] = make_uint4(0u, 0u, 0u, 0u);
            if (t < nt && v < nvec) {
                x.lo[i] = __ldg(reinterpret_cast<const uint4*>(row + (long long)v * HD));
                x.hi[i] = __ldg(reinterpret_cast<const uint4*>(row + (long long)v * HD + HALF));
            }
        }
    };
    Batch next;
    int t = 0, v0 = first + grp;
    load(next, t, v0);
    if (threadIdx.x < nt) {
        const int b = paged_find(p, t0 + threadIdx.x);
        const int pos = paged_pos_of(paged_seq(p, b, fault), t0 + threadIdx.x);
        int page = -1;
        if (pos >= 0) {   // else no sequence's row, or before position 0
            if (rotate && pos >= a.max_seq) atomicOr(fault, (unsigned)AF_FAULT_POSITION);
            else page = paged_page(p, b, pos, fault);
        }
        s_pos[threadIdx.x] = pos;
        s_page[threadIdx.x] = page;
    }
    __syncthreads();
    float4 c[2], sn[2];
    c[0] = c[1] = make_float4(1.f, 1.f, 1.f, 1.f);
    sn[0] = sn[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    long long at = 0, scale_at = 0;   // of the token's first kv head
    __half* q_row = nullptr;
    for (bool new_token = true; t < nt;) {
        const Batch now = next;
        const int tt = t, vv = v0;
        v0 += kWriteBatch * GROUPS;
        if (v0 - grp >= nvec) {
            v0 = first + grp;
            ++t;
        }
        load(next, t, v0);
        const int page = s_page[tt], pos = s_pos[tt];
        const bool first_batch = new_token;
        new_token = t != tt;
        if (page < 0) continue;   // the same for the whole CTA
        if (first_batch) {
            at = paged_at(p, page, pos, 0, HD * KvFormat<FMT>::kBytes);
            scale_at = paged_scale(p, page, pos, 0);
            q_row = a.q_out + (long long)(t0 + tt) * a.NH * HD;
        }
        if (rotate && first_batch) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                c[j] = __ldg(reinterpret_cast<const float4*>(a.cos + (long long)pos * HALF) + 2 * l + j);
                sn[j] = __ldg(reinterpret_cast<const float4*>(a.sin + (long long)pos * HALF) + 2 * l + j);
            }
        }
        const float ca[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w};
        const float sa[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
        for (int i = 0; i < kWriteBatch; ++i) {
            const int v = vv + i * GROUPS;
            if (v - grp >= nvec) break;   // uniform over the warp: the shuffles below take every lane
            const bool on = v < nvec, is_v = v >= a.NH + p.NKV;
            uint4 lo = now.lo[i], hi = now.hi[i];
            __half2* pl = reinterpret_cast<__half2*>(&lo);
            __half2* ph = reinterpret_cast<__half2*>(&hi);
            if (rotate && !is_v) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = __half22float2(pl[j]), y = __half22float2(ph[j]);
                    float2 r0, r1;
                    rope_pair(x.x, y.x, ca[2 * j], sa[2 * j], r0.x, r1.x);
                    rope_pair(x.y, y.y, ca[2 * j + 1], sa[2 * j + 1], r0.y, r1.y);
                    pl[j] = __float22half2_rn(r0);
                    ph[j] = __float22half2_rn(r1);
                }
            }
            const int h = v - a.NH - (is_v ? p.NKV : 0);   // kv head; negative for q
            uint8_t* dst = (is_v ? p.v : p.k) + at + h * (HD * KvFormat<FMT>::kBytes);   // (not used for q)
            if constexpr (FMT == AF_KV_F16) {
                if (on) {
                    __half* out = v < a.NH ? q_row + v * HD : reinterpret_cast<__half*>(dst);
                    *reinterpret_cast<uint4*>(out + 8 * l) = lo;
                    *reinterpret_cast<uint4*>(out + HALF + 8 * l) = hi;
                }
            } else {
                // (NaN does not count)
                __half2 m2 = __hmax2(__habs2(pl[0]), __habs2(ph[0]));
#pragma unroll
                for (int j = 1; j < 4; ++j) m2 = __hmax2(m2, __hmax2(__habs2(pl[j]), __habs2(ph[j])));
                __half m1 = __hmax(__low2half(m2), __high2half(m2));
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) m1 = __hmax(m1, __shfl_xor_sync(0xffffffffu, m1, o));
                const float amax = m1 == m1 ? __half2float(m1) : 0.f;
                if (on && v < a.NH) {
                    __half* out = q_row + v * HD;
                    *reinterpret_cast<uint4*>(out + 8 * l) = lo;
                    *reinterpret_cast<uint4*>(out + HALF + 8 * l) = hi;
                } else if (on) {
                    const __half sc = kv_scale<FMT>(amax);
                    const float f = __half2float(sc), rcp = __frcp_rn(f);
                    *reinterpret_cast<uint2*>(dst + 8 * l) =
                        make_uint2(kv_pack4<FMT>(pl[0], pl[1], f, rcp), kv_pack4<FMT>(pl[2], pl[3], f, rcp));
                    *reinterpret_cast<uint2*>(dst + HALF + 8 * l) =
                        make_uint2(kv_pack4<FMT>(ph[0], ph[1], f, rcp), kv_pack4<FMT>(ph[2], ph[3], f, rcp));
                    if (l == 0) (is_v ? p.vs : p.ks)[scale_at + h] = sc;
                }
            }
        }
    }
}

// ----------------------------------------------------------------- read
// Rows of positions -> contiguous FP16.  A CTA takes kReadRows rows; each
// thread moves 16-byte pieces (one piece of an 8-bit cache makes two of FP16).
// Bound by DRAM: codes in, FP16 out.
constexpr int kReadThreads = 256;
constexpr int kReadRows = 8;
constexpr int kReadBatch = 4;

template <int FMT, int HD>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const Paged p, __half* __restrict__ k_out,
                                                                  __half* __restrict__ v_out, unsigned* fault) {
    __shared__ long long s_at[kReadRows];    // page * 2^32 + slot of each row; -1: zeros; -2: not ours
    const int t0 = blockIdx.x * kReadRows;
    if (threadIdx.x < kReadRows) {
        const int t = t0 + threadIdx.x;
        long long at = -2;
        if (t < p.n_tokens) {
            const int b = paged_find(p, t);
            const PagedSeq s = paged_seq(p, b, fault);
            const int pos = paged_pos_of(s, t);
            if (pos > INT_MIN) {
                const int page = pos < 0 ? -1 : paged_page(p, b, pos, fault);
                at = page < 0 ? -1 : ((long long)page << 32) | paged_slot_of(pos, p.page_shift);
            }
        }
        s_at[threadIdx.x] = at;
    }
    __syncthreads();
    constexpr int PER = HD * KvFormat<FMT>::kBytes / 16;   // pieces of one vector
    const int pieces = p.NKV * PER;                        // of one row of K (or V)
    const int total = kReadRows * 2 * pieces;
    for (int i0 = threadIdx.x; i0 < total; i0 += kReadBatch * kReadThreads) {
        uint4 x[kReadBatch];
        __half sc[kReadBatch];
#pragma unroll
        for (int j = 0; j < kReadBatch; ++j) {
            const int i = i0 + j * kReadThreads;
            x[j] = make_uint4(0u, 0u, 0u, 0u);
            sc[j] = __float2half_rn(0.f);
            if (i >= total) continue;
            const int r = i / (2 * pieces), w = i % (2 * pieces), piece = w % pieces;
            const bool is_v = w >= pieces;
            const long long at = s_at[r];
            if (at < 0) continue;
            const int page = (int)(at >> 32), slot = (int)(at & 0xffffffff);
            x[j] = ldg_stream((is_v ? p.v : p.k) + paged_at(p, page, slot, 0, HD * KvFormat<FMT>::kBytes) + piece * 16);
            if constexpr (FMT != AF_KV_F16) sc[j] = __ldg((is_v ? p.vs : p.ks) + paged_scale(p, page, slot, piece / PER));
        }
#pragma unroll
        for (int j = 0; j < kReadBatch; ++j) {
            const int i = i0 + j * kReadThreads;
            if (i >= total) continue;
            const int r = i / (2 * pieces), w = i % (2 * pieces), piece = w % pieces;
            if (s_at[r] == -2) continue;
            __half* out = (w >= pieces ? v_out : k_out) + (long long)(t0 + r) * p.NKV * HD +
                          (long long)piece * (16 / KvFormat<FMT>::kBytes);
            if constexpr (FMT == AF_KV_F16) {
                *reinterpret_cast<uint4*>(out) = x[j];
            } else {
                const __half2 s2 = __half2half2(sc[j]);
                uint32_t o[8];
                const uint32_t in[4] = {x[j].x, x[j].y, x[j].z, x[j].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    kv_unpack4<FMT>(in[q], o[2 * q], o[2 * q + 1]);
                    o[2 * q] = mul_half2(o[2 * q], s2);
                    o[2 * q + 1] = mul_half2(o[2 * q + 1], s2);
                }
                reinterpret_cast<uint4*>(out)[0] = make_uint4(o[0], o[1], o[2], o[3]);
                reinterpret_cast<uint4*>(out)[1] = make_uint4(o[4], o[5], o[6], o[7]);
            }
        }
    }
}

}  // namespace

namespace af {

unsigned* paged_fault_word(cudaError_t* err) {
    static std::atomic<unsigned*> word[kMaxDevices];
    int dev = 0;
    *err = cudaGetDevice(&dev);
    if (*err != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
    unsigned* w = word[dev].load(std::memory_order_acquire);
    if (w == nullptr) {
        void* ptr = nullptr;
        *err = cudaGetSymbolAddress(&ptr, g_paged_faults);
        if (*err != cudaSuccess) return nullptr;
        w = static_cast<unsigned*>(ptr);
        word[dev].store(w, std::memory_order_release);
    }
    return w;
}

unsigned paged_faults(bool clear, cudaError_t* err) {
    unsigned v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_paged_faults, sizeof(v));
    if (e == cudaSuccess && clear && v != 0) {
        const unsigned z = 0;
        e = cudaMemcpyToSymbol(g_paged_faults, &z, sizeof(z));
    }
    *err = e;
    return v;
}

af_status paged_args(const af_paged_kv* kv, const af_paged_batch* batch, Paged* out) {
    if (kv == nullptr || batch == nullptr) return AF_ERR_INVALID;
    if (kv->format != AF_KV_F16 && kv->format != AF_KV_FP8_E4M3 && kv->format != AF_KV_INT8) return AF_ERR_INVALID;
    if (kv->head_dim != 64 && kv->head_dim != 128) return AF_ERR_UNSUPPORTED;
    if (kv->n_pages < 0 || kv->n_kv_heads < 1 || kv->n_kv_heads > 1024) return AF_ERR_INVALID;
    const int ps = kv->page_size;
    if (ps < kPagedMinPage || ps > kPagedMaxPage || (ps & (ps - 1)) != 0) return AF_ERR_UNSUPPORTED;
    if (batch->n_seqs < 0 || batch->n_tokens < 0 || batch->max_pages < 0) return AF_ERR_INVALID;
    const bool quant = kv->format != AF_KV_F16;
    if (!quant && (kv->k_scale != nullptr || kv->v_scale != nullptr)) return AF_ERR_INVALID;
    const long long esz = quant ? 1 : 2;
    const long long row = (long long)kv->n_kv_heads * kv->head_dim;
    if (kv->page_stride < ps * row || (kv->page_stride * esz) % 16 != 0) return AF_ERR_INVALID;
    if (quant && kv->scale_stride < (long long)ps * kv->n_kv_heads) return AF_ERR_INVALID;
    if (batch->table_stride < batch->max_pages) return AF_ERR_INVALID;
    if (batch->n_seqs > 0 && batch->n_tokens > 0) {
        if (kv->k == nullptr || kv->v == nullptr || !aligned(kv->k, 16) || !aligned(kv->v, 16)) return AF_ERR_INVALID;
        if (quant && (kv->k_scale == nullptr || kv->v_scale == nullptr || !aligned(kv->k_scale, 2) ||
                      !aligned(kv->v_scale, 2)))
            return AF_ERR_INVALID;
        if (batch->cu_rows == nullptr || batch->kv_len == nullptr || !aligned(batch->cu_rows, 4) ||
            !aligned(batch->kv_len, 4))
            return AF_ERR_INVALID;
        if (batch->max_pages > 0 && (batch->block_table == nullptr || !aligned(batch->block_table, 4)))
            return AF_ERR_INVALID;
    }
    int shift = 0;
    while ((1 << shift) < ps) ++shift;
    out->k = static_cast<uint8_t*>(kv->k);
    out->v = static_cast<uint8_t*>(kv->v);
    out->ks = static_cast<__half*>(kv->k_scale);
    out->vs = static_cast<__half*>(kv->v_scale);
    out->page_bytes = kv->page_stride * esz;
    out->scale_stride = kv->scale_stride;
    out->cu = batch->cu_rows;
    out->len = batch->kv_len;
    out->table = batch->block_table;
    out->table_stride = batch->table_stride;
    out->n_pages = kv->n_pages;
    out->page_shift = shift;
    out->NKV = kv->n_kv_heads;
    out->n_seqs = batch->n_seqs;
    out->n_tokens = batch->n_tokens;
    out->max_pages = batch->max_pages;
    return AF_OK;
}

// Whether [a, a + n) and [b, b + m) share a byte.
static bool overlap(const void* a, long long n, const void* b, long long m) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)m && y < x + (uintptr_t)n;
}

// Calls f<FMT, HD>() for the cache's format and head size (checked by paged_args).
template <class F>
static void paged_dispatch(const af_paged_kv* kv, F&& f) {
    auto hd = [&](auto fmt) {
        if (kv->head_dim == 128) f(fmt, std::integral_constant<int, 128>());
        else f(fmt, std::integral_constant<int, 64>());
    };
    if (kv->format == AF_KV_F16) hd(std::integral_constant<int, AF_KV_F16>());
    else if (kv->format == AF_KV_FP8_E4M3) hd(std::integral_constant<int, AF_KV_FP8_E4M3>());
    else hd(std::integral_constant<int, AF_KV_INT8>());
}

}  // namespace af

extern "C" af_status af_paged_kv_write(const af_paged_kv* kv, const af_paged_batch* batch, const void* qkv,
                                       int64_t qkv_stride, int n_heads, const float* cos_tab, const float* sin_tab,
                                       int max_seq, void* q_out, void* stream) {
    Paged p;
    const af_status st = paged_args(kv, batch, &p);
    if (st != AF_OK) return st;
    if (n_heads < 0 || n_heads > 65535 || (cos_tab == nullptr) != (sin_tab == nullptr)) return AF_ERR_INVALID;
    if (qkv_stride < (int64_t)(n_heads + 2 * p.NKV) * kv->head_dim || qkv_stride % 8 != 0) return AF_ERR_INVALID;
    if (cos_tab != nullptr && (max_seq < 1 || !aligned(cos_tab, 16) || !aligned(sin_tab, 16))) return AF_ERR_INVALID;
    if (p.n_seqs == 0 || p.n_tokens == 0) return AF_OK;
    if (qkv == nullptr || !aligned(qkv, 16)) return AF_ERR_INVALID;
    const long long row = (long long)(n_heads + 2 * p.NKV) * kv->head_dim;
    if (cos_tab != nullptr && n_heads > 0 &&
        (q_out == nullptr || !aligned(q_out, 16) ||
         overlap(q_out, 2LL * p.n_tokens * n_heads * kv->head_dim, qkv, 2 * ((p.n_tokens - 1) * qkv_stride + row))))
        return AF_ERR_INVALID;
    cudaError_t e;
    unsigned* fault = paged_fault_word(&e);
    if (fault == nullptr) return cuda_fail(e, "af_paged_kv_write");
    // tokens of a CTA: one while that leaves SMs idle, more once there are several CTAs for each
    const int tokens = std::max(1, std::min(kWriteTokens, p.n_tokens / (8 * std::max(1, device_sm_count()))));
    const WriteArgs a{static_cast<const __half*>(qkv), qkv_stride, cos_tab, sin_tab, static_cast<__half*>(q_out),
                      n_heads, max_seq, tokens};
    const unsigned grid = (unsigned)(((long long)p.n_tokens + tokens - 1) / tokens);
    paged_dispatch(kv, [&](auto fmt, auto hd) {
        paged_write_kernel<decltype(fmt)::value, decltype(hd)::value>
            <<<grid, kWriteThreads, 0, static_cast<cudaStream_t>(stream)>>>(p, a, fault);
    });
    e = cudaGetLastError();
    return e == cudaSuccess ? AF_OK : cuda_fail(e, "paged_write_kernel");
}

extern "C" af_status af_paged_kv_read(const af_paged_kv* kv, const af_paged_batch* batch, void* k_out, void* v_out,
                                      void* stream) {
    Paged p;
    const af_status st = paged_args(kv, batch, &p);
    if (st != AF_OK) return st;
    if (p.n_seqs == 0 || p.n_tokens == 0) return AF_OK;
    const long long bytes = 2LL * p.n_tokens * p.NKV * kv->head_dim;
    if (k_out == nullptr || v_out == nullptr || !aligned(k_out, 16) || !aligned(v_out, 16) ||
        overlap(k_out, bytes, v_out, bytes))
        return AF_ERR_INVALID;
    cudaError_t e;
    unsigned* fault = paged_fault_word(&e);
    if (fault == nullptr) return cuda_fail(e, "af_paged_kv_read");
    const unsigned grid = (unsigned)(((long long)p.n_tokens + kReadRows - 1) / kReadRows);
    paged_dispatch(kv, [&](auto fmt, auto hd) {
        paged_read_kernel<decltype(fmt)::value, decltype(hd)::value>
            <<<grid, kReadThreads, 0, static_cast<cudaStream_t>(stream)>>>(
                p, static_cast<__half*>(k_out), static_cast<__half*>(v_out), fault);
    });
    e = cudaGetLastError();
    return e == cudaSuccess ? AF_OK : cuda_fail(e, "paged_read_kernel");
}

namespace {

// Which kernels an attention call runs.  Which sequences each takes is a matter of their rows (new tokens x query heads
// per kv head), which only the device knows; the host's bounds say which kernels can have work.
struct AttnPlan {
    bool few, chunk;    // sequences of at most kFewRows rows; longer ones
    int few_rows;       // bound on the rows of the former
    int skip_rows;      // the chunk kernel leaves sequences of at most these to the other
    int kv;             // bound on the cached positions
};
AttnPlan attn_plan(const Paged& p, int n_heads, int max_rows, int max_kv) {
    AttnPlan x;
    x.kv = paged_kv_bound(max_kv, p.max_pages, p.page_shift);
    const int q = max_rows > 0 ? std::min(max_rows, p.n_tokens) : p.n_tokens;
    const long long rows = (long long)q * (n_heads / p.NKV);
    const bool even = (long long)q * p.n_seqs <= p.n_tokens;   // every sequence as long as the bound: none is short
    x.chunk = rows > kFewRows;
    x.few = !x.chunk || !even;
    x.few_rows = (int)std::min<long long>(rows, kFewRows);
    x.skip_rows = even ? 0 : kFewRows;
    return x;
}

af_status attn_args(const af_paged_kv* kv, const af_paged_batch* batch, int n_heads, int max_rows, int max_kv, Paged* p) {
    const af_status st = paged_args(kv, batch, p);
    if (st != AF_OK) return st;
    if (n_heads < 1 || n_heads > 65535 || n_heads % p->NKV != 0 || max_rows < 0 || max_kv < 0) return AF_ERR_INVALID;
    return (long long)p->n_tokens * (n_heads / p->NKV) > INT_MAX ? AF_ERR_UNSUPPORTED : AF_OK;
}

}  // namespace

extern "C" size_t af_paged_attention_workspace_bytes(const af_paged_kv* kv, const af_paged_batch* batch, int n_heads,
                                                     int max_rows, int max_kv) {
    Paged p;
    if (attn_args(kv, batch, n_heads, max_rows, max_kv, &p) != AF_OK || p.n_seqs == 0 || p.n_tokens == 0) return 0;
    const AttnPlan x = attn_plan(p, n_heads, max_rows, max_kv);
    return x.few ? paged_few_workspace(kv->format, kv->head_dim, p, x.few_rows, x.kv) : 0;
}

extern "C" af_status af_paged_attention(const af_paged_kv* kv, const af_paged_batch* batch, const void* q,
                                        int64_t q_stride, int n_heads, float scale, int max_rows, int max_kv,
                                        void* out, void* workspace, size_t workspace_bytes, void* stream) {
    Paged p;
    const af_status st = attn_args(kv, batch, n_heads, max_rows, max_kv, &p);
    if (st != AF_OK) return st;
    if (q_stride < (int64_t)n_heads * kv->head_dim || q_stride % 8 != 0) return AF_ERR_INVALID;
    if (!(scale > 0.f) || !std::isfinite(scale) || !aligned(workspace, 16)) return AF_ERR_INVALID;
    if (p.n_seqs == 0 || p.n_tokens == 0) return AF_OK;
    const long long row = (long long)n_heads * kv->head_dim;
    if (q == nullptr || out == nullptr || !aligned(q, 16) || !aligned(out, 16) ||
        overlap(out, 2 * p.n_tokens * row, q, 2 * ((p.n_tokens - 1) * q_stride + row)))
        return AF_ERR_INVALID;
    cudaError_t e;
    unsigned* fault = paged_fault_word(&e);
    if (fault == nullptr) return cuda_fail(e, "af_paged_attention");
    const AttnPlan x = attn_plan(p, n_heads, max_rows, max_kv);
    const cudaStream_t cs = static_cast<cudaStream_t>(stream);
    // the long sequences first: the short ones' CTAs fill the SMs that their last wave leaves idle
    if (x.chunk)
        e = paged_chunk_launch(kv->format, kv->head_dim, p, q, q_stride, n_heads, scale, x.skip_rows, x.kv, out, fault, cs);
    if (x.few && e == cudaSuccess)
        e = paged_few_launch(kv->format, kv->head_dim, p, q, q_stride, n_heads, scale, x.few_rows, x.chunk, x.kv, out,
                             workspace, workspace_bytes, fault, cs);
    return e == cudaSuccess ? AF_OK : cuda_fail(e, "af_paged_attention");
}

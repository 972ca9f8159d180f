// af_paged.cuh -- what the kernels over a paged KV cache share: the cache and the
// batch as they see them, the checks that keep every access inside the pool
// whatever the device arrays hold, and the cache formats' codes.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <cstdint>

#include "af_common.cuh"
#include "af_internal.h"
#include "af_paged_index.h"

namespace af {

constexpr int kPagedMinPage = 8, kPagedMaxPage = 256;

// The cache and the batch, by value, as a kernel argument.
struct Paged {
    uint8_t *k, *v;              // pages [n_pages][page][NKV][HD]
    __half *ks, *vs;             // scales [n_pages][page][NKV] (8-bit formats)
    long long page_bytes;        // from one page to the next
    long long scale_stride;      // scales from one page to the next
    const int *cu, *len, *table;
    long long table_stride;
    int n_pages, page_shift, NKV;
    int n_seqs, n_tokens, max_pages;
};

// Fault bits of the paged operators (af_paged.cu), through a pointer: the
// kernels live in several translation units.
unsigned* paged_fault_word(cudaError_t* err);

// Sequence b; a bad one sets the fault bit and has no rows.
__device__ __forceinline__ PagedSeq paged_seq(const Paged& p, int b, unsigned* fault) {
    const PagedSeq s = paged_seq_of(__ldg(p.cu + b), __ldg(p.cu + b + 1), __ldg(p.len + b), p.n_tokens, p.max_pages,
                                    p.page_shift);
    if (s.bad) atomicOr(fault, (unsigned)AF_FAULT_PAGED);
    return s;
}

// The sequence whose rows hold row t: the last b with cu[b] <= t (empty
// sequences share their offset with the next one).  Not checked: paged_seq is.
__device__ __forceinline__ int paged_find(const Paged& p, int t) {
    int lo = 0, hi = p.n_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldg(p.cu + mid) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Page of position pos of sequence b; -1 (and the fault bit) where the table's
// entry is not a page of the pool.
__device__ __forceinline__ int paged_page(const Paged& p, int b, int pos, unsigned* fault) {
    const int page = __ldg(p.table + paged_table_at(b, p.table_stride, pos, p.page_shift));
    if (paged_page_ok(page, p.n_pages)) return page;
    atomicOr(fault, (unsigned)AF_FAULT_PAGED);
    return -1;
}
// Byte offset of a head vector of the pool, index of its scale.
__device__ __forceinline__ long long paged_at(const Paged& p, int page, int pos, int head, int vector_bytes) {
    return paged_vector_at(page, p.page_bytes, paged_slot_of(pos, p.page_shift), p.NKV, head, vector_bytes);
}
__device__ __forceinline__ long long paged_scale(const Paged& p, int page, int pos, int head) {
    return paged_scale_at(page, p.scale_stride, paged_slot_of(pos, p.page_shift), p.NKV, head);
}

// ---- formats ----
template <int FMT>
struct KvFormat;
template <>
struct KvFormat<AF_KV_F16> {
    static constexpr int kBytes = 2;
};
// 8-bit codes: value = code * scale.  kScaleMax is the largest FP16 scale whose
// product with the largest code is a finite FP16 value.
template <>
struct KvFormat<AF_KV_FP8_E4M3> {
    static constexpr int kBytes = 1;
    static constexpr float kCodeMax = 448.f, kScaleMax = 146.125f;
};
template <>
struct KvFormat<AF_KV_INT8> {
    static constexpr int kBytes = 1;
    static constexpr float kCodeMax = 127.f, kScaleMax = 515.5f;
};

// Four codes (one word, lowest address first) -> four FP16 values in two words, exactly.
// E4M3 by the packed conversion.  INT8: byte b ^ 0x80 as the mantissa of 1024
// gives 1024 + b + 128 exactly; subtracting 1152 leaves b.
template <int FMT>
__device__ __forceinline__ void kv_unpack4(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if constexpr (FMT == AF_KV_FP8_E4M3) {
        lo = e4m3x2_lo(w);
        hi = e4m3x2_hi(w);
    } else {
        w ^= 0x80808080u;
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 off = __float2half2_rn(1152.f);
        const __half2 ra = __hsub2(*reinterpret_cast<const __half2*>(&a), off);
        const __half2 rb = __hsub2(*reinterpret_cast<const __half2*>(&b), off);
        lo = *reinterpret_cast<const uint32_t*>(&ra);
        hi = *reinterpret_cast<const uint32_t*>(&rb);
    }
}
// Two FP16 values times a pair of FP16 scales, one rounding each.
__device__ __forceinline__ uint32_t mul_half2(uint32_t v, __half2 s) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&v), s);
    return *reinterpret_cast<const uint32_t*>(&r);
}

// A scale = power * rest, exactly, power a power of two whose product with every code is an FP16 value (down to FP16's
// subnormals: INT8's codes are whole numbers, E4M3's multiples of 2^-9) and at most 2^MAX.  rest is in [1, 2), below
// that where the power is the smallest, above where it is the largest; a scale that is not finite is all rest.
struct KvScaleParts {
    __half power;
    float rest;
};
template <int FMT, int MAX>
__device__ __forceinline__ KvScaleParts kv_split_scale(float scale) {
    constexpr int MIN = FMT == AF_KV_INT8 ? -24 : -15;
    int e = (int)((__float_as_uint(scale) >> 23) & 255u) - 127;   // (an FP16 value is a normal FP32 one, or 0)
    e = e > 15 ? 0 : min(max(e, MIN), MAX);
    return {__float2half_rn(__uint_as_float((uint32_t)(e + 127) << 23)), scale * __uint_as_float((uint32_t)(127 - e) << 23)};
}

// The scale of a vector whose largest magnitude is amax: the smallest FP16 value
// that brings it to at most the largest code (rounded up, so that no element
// saturates however small the scale), 1 for a vector of zeros.  NaN elements do
// not count; an infinity takes the largest scale.
template <int FMT>
__device__ __forceinline__ __half kv_scale(float amax) {
    if (amax == 0.f) return __float2half_rn(1.f);
    const __half s = __float2half_ru(__fdiv_rn(amax, KvFormat<FMT>::kCodeMax));
    return __hmin(s, __float2half_rn(KvFormat<FMT>::kScaleMax));
}
// Four values -> four codes: round to nearest even of x / scale, saturating.  x and the scale are FP16 values, and the
// quotient matters only to a code's half step (9 bits at most): unless it is such a border itself it is 2^-20 away from
// one, relatively, so x * rcp would do; and where it is one, the residual's correction makes it exact (rcp = 1 / scale
// correctly rounded, q = x rcp (1 + 2^-23) at worst, and q + (x - q scale) rcp is then exact to 2^-46 before its
// rounding).  Infinities count as the largest FP16 value; NaN stays (INT8: 0).
template <int FMT>
__device__ __forceinline__ uint32_t kv_pack4(__half2 h0, __half2 h1, float scale, float rcp) {
    const __half2 h[2] = {h0, h1};
    const __half2 top = __float2half2_rn(65504.f);
    float y[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 x = __half22float2(__hmin2_nan(__hmax2_nan(h[i], __hneg2(top)), top));
        const float q0 = x.x * rcp, q1 = x.y * rcp;
        y[2 * i] = fmaf(fmaf(-q0, scale, x.x), rcp, q0);
        y[2 * i + 1] = fmaf(fmaf(-q1, scale, x.y), rcp, q1);
    }
    if constexpr (FMT == AF_KV_FP8_E4M3) {
        const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t b = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
        // the correction of a quotient of -0 is +0: the sign comes from x
        const uint32_t sign = __byte_perm(*reinterpret_cast<const uint32_t*>(&h[0]), *reinterpret_cast<const uint32_t*>(&h[1]), 0x7531);
        return a | (b << 16) | (sign & 0x80808080u);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // + 1.5 * 2^23 rounds to the nearest integer and leaves it in the low bits
            const float c = y[i] == y[i] ? fminf(fmaxf(y[i], -127.f), 127.f) : 0.f;
            w[i] = __float_as_uint(c + 12582912.f);
        }
        return __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
    }
}

// ---- V at positions that some row of a tile does not see ----
// Such a row's weight is zero, but zero times an infinity or NaN is NaN: both attention kernels put zeros in their
// place in the tile, and add them back to the rows that do see them.
// V's element as the attention sees it.
template <int FMT, int HD>
__device__ float v_value(const Paged& p, int b, int pos, int kvh, int d, unsigned* fault) {
    const int page = paged_page(p, b, pos, fault);
    if (page < 0) return 0.f;
    const uint8_t* at = p.v + paged_at(p, page, pos, kvh, HD * KvFormat<FMT>::kBytes);
    if constexpr (FMT == AF_KV_F16) return __half2float(reinterpret_cast<const __half*>(at)[d]);
    const float s = __half2float(p.vs[paged_scale(p, page, pos, kvh)]);
    if constexpr (FMT == AF_KV_INT8) return (float)reinterpret_cast<const int8_t*>(at)[d] * s;
    return (float)reinterpret_cast<const __nv_fp8_e4m3*>(at)[d] * s;
}
// Puts zeros in the place of infinities and NaN in a pair of FP16 values; whether there were any.
__device__ __forceinline__ bool mend_half2(uint32_t& v) {
    const bool lo = (v & 0x7c00u) == 0x7c00u, hi = (v & 0x7c000000u) == 0x7c000000u;
    if (lo) v &= 0xffff0000u;
    if (hi) v &= 0x0000ffffu;
    return lo | hi;
}
__device__ __forceinline__ bool mend_chunk(uint4& v) {
    const bool a = mend_half2(v.x), b = mend_half2(v.y), c = mend_half2(v.z), d = mend_half2(v.w);
    return a | b | c | d;
}


// ---- host side (af_paged.cu) ----
af_status paged_args(const af_paged_kv* kv, const af_paged_batch* batch, Paged* out);
// The attention of few rows (af_paged_few.cu): every sequence of at most 8 (rows_bound <= 8) or kFewRows rows (tokens x
// query heads per kv head).  behind: the tensor-core kernel was launched just before and takes the others; this one may
// begin while it still runs (they touch different rows).  Else sequences of more rows are recorded as a fault.
constexpr int kFewRows = 16;
size_t paged_few_workspace(int format, int head_dim, const Paged& p, int rows_bound, int max_kv);
cudaError_t paged_few_launch(int format, int head_dim, const Paged& p, const void* q, long long q_stride, int n_heads,
                             float scale, int rows_bound, bool behind, int max_kv, void* out, void* workspace,
                             size_t workspace_bytes, unsigned* fault, cudaStream_t st);
// The tensor-core attention (af_paged_tc.cu) over every sequence of more than
// skip_rows rows (tokens x query heads per kv head).
cudaError_t paged_chunk_launch(int format, int head_dim, const Paged& p, const void* q, long long q_stride, int n_heads,
                               float scale, int skip_rows, int max_kv, void* out, unsigned* fault, cudaStream_t st);

}  // namespace af

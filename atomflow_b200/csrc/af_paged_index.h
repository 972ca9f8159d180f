// af_paged_index.h -- the index arithmetic of the paged KV cache, in plain C++ for
// host and device: what keeps every access of the paged kernels inside the
// buffers whatever the device arrays hold, and the 64-bit offsets.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define AF_HD __host__ __device__ __forceinline__
#else
#define AF_HD inline
#endif

namespace af {

// One sequence: its rows [row0, row0 + q) and its cached positions [0, kv).
struct PagedSeq {
    int row0, q, kv;
    bool bad;
};
// From the sequence's two row offsets and its length.  Rows outside [0, n_tokens),
// decreasing offsets, a negative length or one beyond max_pages pages or 2^30
// (so that a position plus a tile fits in an int): a bad sequence, without rows.
AF_HD PagedSeq paged_seq_of(int s, int e, int kv, int n_tokens, int max_pages, int page_shift) {
    if (s < 0 || e < s || e > n_tokens || kv < 0 || kv > (1 << 30) || (int64_t)kv > ((int64_t)max_pages << page_shift))
        return {0, 0, 0, true};
    return {s, e - s, kv, false};
}
// Position of the sequence's row t (of all rows); negative: before the cache.
// INT_MIN where t is none of its rows.
AF_HD int paged_pos_of(const PagedSeq& s, int t) {
    if (t < s.row0 || t - s.row0 >= s.q) return -2147483647 - 1;
    return s.kv - s.q + (t - s.row0);
}
AF_HD bool paged_page_ok(int page, int n_pages) { return page >= 0 && page < n_pages; }
// A position's row of NKV vectors in its page, and a head vector's offsets.
AF_HD int paged_slot_of(int pos, int page_shift) { return pos & ((1 << page_shift) - 1); }
AF_HD int64_t paged_table_at(int b, int64_t table_stride, int pos, int page_shift) {
    return (int64_t)b * table_stride + (pos >> page_shift);
}
AF_HD int64_t paged_vector_at(int page, int64_t page_bytes, int slot, int nkv, int head, int vector_bytes) {
    return (int64_t)page * page_bytes + ((int64_t)slot * nkv + head) * vector_bytes;
}
AF_HD int64_t paged_scale_at(int page, int64_t scale_stride, int slot, int nkv, int head) {
    return (int64_t)page * scale_stride + (int64_t)slot * nkv + head;
}

}  // namespace af

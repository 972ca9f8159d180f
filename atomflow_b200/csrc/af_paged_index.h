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
constexpr int kPagedMaxKv = 1 << 30;   // of a sequence, so that a position plus a tile fits in an int
// From the sequence's two row offsets and its length.  Rows outside [0, n_tokens),
// decreasing offsets, a negative length or one beyond max_pages pages or
// kPagedMaxKv: a bad sequence, without rows.
AF_HD PagedSeq paged_seq_of(int s, int e, int kv, int n_tokens, int max_pages, int page_shift) {
    if (s < 0 || e < s || e > n_tokens || kv < 0 || kv > kPagedMaxKv || (int64_t)kv > ((int64_t)max_pages << page_shift))
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


// What a sequence's cached positions are at most: the caller's bound (0: none), the table, the largest length.
inline int paged_kv_bound(int max_kv, int max_pages, int page_shift) {
    int64_t n = (int64_t)max_pages << page_shift;
    if (max_kv > 0 && max_kv < n) n = max_kv;
    return n < kPagedMaxKv ? (int)n : kPagedMaxKv;
}

// Over how many CTAs (a power of two) the chunk kernel splits the positions of its work items, of at most `tiles` tiles
// each, on a GPU of `sms` SMs (0 or less: not known): as many as shorten the whole, waves of CTAs x (tiles of each + what a
// CTA costs beside its tiles, about 3 tiles' time alone and 6 in a cluster that merges).  Clusters leave SMs out: of 148,
// cudaOccupancyMaxActiveClusters gives 148, 148, 132 and 120 to clusters of 1, 2, 4 and 8 such CTAs; a GPU too small for
// a size does not use it.  (128 new tokens x 4 over 8192, 16 items: 8 CTAs, 16 clusters for 15 places, 64 us; 4 CTAs 47 us.)
constexpr int kPagedMaxSplit = 8;
inline int paged_chunk_split(int64_t items, int tiles, int sms) {
    if (sms < 1) sms = 1;
    const int place[4] = {sms, sms / 2 * 2, sms * 33 / 148 * 4, sms * 15 / 148 * 8};
    int split = 1;
    double best = 1e300;
    for (int i = 0; 1 << i <= kPagedMaxSplit && (i == 0 || tiles >= 4 << i); ++i) {   // four tiles per CTA at least
        if (place[i] == 0) continue;
        const int64_t ctas = items << i, waves = (ctas + place[i] - 1) / place[i];
        const double cost = (double)waves * ((double)tiles / (1 << i) + (i == 0 ? 3. : 6.));
        if (cost < best) {
            best = cost;
            split = 1 << i;
        }
    }
    return split;
}

}  // namespace af

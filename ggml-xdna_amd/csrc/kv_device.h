// What the paged KV cache's kernels share: its layout, the checked view of a
// batch's sequences, and the prefix sums by which a workgroup finds its work.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "zest/kv.h"

namespace zest {

constexpr int KV_MAX_SEQS = 4096;

struct kv_pages {
    uint8_t * pool;
    int64_t page_bytes;
    int32_t pages, kv_heads, page_shift;  // tokens a page: 1 << page_shift
};

struct kv_batch {
    const int32_t * tables, * lens, * starts, * slots;
    int64_t rows;
    int32_t seqs, table_rows, table_cols, max_new, max_len;
    uint32_t * bad;
};

__device__ inline void report(uint32_t * bad) {
    if (bad) atomicOr(bad, 1u);
}

// One sequence as the device tensors give it: n = 0 where it has no new tokens
// or its numbers do not fit the bounds.
struct kv_seq {
    int32_t row0, n, len, slot;
};

__device__ inline kv_seq load_seq(const kv_batch & a, int b, int page_shift, bool & bad) {
    kv_seq s{a.starts[b], 0, 0, a.slots ? a.slots[b] : b};
    const int32_t end = a.starts[b + 1];
    if (end == s.row0) return s;
    if (s.row0 < 0 || end < s.row0 || end > a.rows || end - s.row0 > a.max_new || (uint32_t) s.slot >= (uint32_t) a.table_rows) {
        bad = true;
        return s;
    }
    s.len = a.lens[s.slot];
    if (s.len < 0 || s.len > a.max_len || s.len > ((int64_t) a.table_cols << page_shift)) {
        bad = true;
        s.len = 0;
        return s;
    }
    s.n = end - s.row0;
    return s;
}

// prefix[b] = sum of cost(sequence) over the sequences before b, for b = 0 ..
// seqs, in shared memory: every thread sums a run of sequences, a wave's sums
// are scanned by lane exchanges and the waves' by every thread. All threads of
// the workgroup (a multiple of 64, at most 1024) call it; it ends in a barrier.
template <typename Cost>
__device__ inline void prefix_over_seqs(const kv_batch & a, int page_shift, int32_t * prefix, Cost cost) {
    __shared__ int32_t wave_sum[16];
    const int t = threadIdx.x, threads = blockDim.x, lane = t & 63;
    const int run = (a.seqs + threads - 1) / threads, first = min(t * run, a.seqs), last = min(first + run, a.seqs);
    bool bad = false;
    int32_t sum = 0;
    for (int b = first; b < last; b++) {
        const int32_t c = cost(load_seq(a, b, page_shift, bad));
        prefix[b + 1] = c;
        sum += c;
    }
    int32_t scan = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t v = __shfl_up(scan, off);
        if (lane >= off) scan += v;
    }
    if (lane == 63) wave_sum[t >> 6] = scan;
    __syncthreads();
    int32_t before = scan - sum;
    for (int w = 0; w < (t >> 6); w++) before += wave_sum[w];
    if (t == 0) prefix[0] = 0;
    for (int b = first; b < last; b++) prefix[b + 1] = before += prefix[b + 1];
    if (bad && blockIdx.x == 0) report(a.bad);
    __syncthreads();
}

// The sequence whose run of the prefix sums holds u (u < prefix[seqs]).
__device__ inline int seq_of(const int32_t * prefix, int seqs, int32_t u) {
    int lo = 0, hi = seqs;  // prefix[lo] <= u < prefix[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (prefix[mid] <= u) lo = mid;
        else hi = mid;
    }
    return lo;
}

inline int kv_page_shift(int page_tokens) { return page_tokens > 0 ? __builtin_ctz((unsigned) page_tokens) : 0; }

inline kv_pages kv_pages_of(const zest_kv_cache * c) {
    return {(uint8_t *) c->pool, (int64_t) zest_kv_page_bytes(c), (int32_t) c->pages, c->kv_heads, kv_page_shift(c->page_tokens)};
}

inline kv_batch kv_batch_of(const zest_kv_batch * b, uint32_t * bad) {
    return {b->tables, b->lens, b->starts, b->slots, b->rows, b->seqs, b->table_rows, b->table_cols, b->max_new, b->max_len, bad};
}

// The host checks every call makes of its cache and batch (zest_status).
int kv_check_cache(const zest_kv_cache * c, const char * what);
int kv_check_batch(const zest_kv_cache * c, const zest_kv_batch * b, const char * what);
int kv_check_rows(int type, const void * p, int64_t ld, int64_t width, const char * what, const char * name);

// Bytes of a value of an F32, F16 or BF16 tensor, 0 for other types.
inline int kv_type_bytes(int type) {
    return type == ZEST_TYPE_F32 ? 4 : type == ZEST_TYPE_F16 || type == ZEST_TYPE_BF16 ? 2 : 0;
}

} // namespace zest

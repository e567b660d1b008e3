// What the paged KV cache's kernels share: its layout, the checked view of a
// batch's sequences, and how a workgroup finds its work among them.
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
    const bool named = (uint32_t) s.slot < (uint32_t) a.table_rows;
    const int32_t len = a.lens[named ? s.slot : 0];  // requested with the starts, not after them
    if (end == s.row0) return s;
    if (!named || s.row0 < 0 || end < s.row0 || end > a.rows || end - s.row0 > a.max_new || len < 0 || len > a.max_len ||
        len > ((int64_t) a.table_cols << page_shift)) {
        bad = true;
        return s;
    }
    s.n = end - s.row0;
    s.len = len;
    return s;
}

// Sequences that a kernel before has looked at: checked, and each with its own place
// in the tables (slot is the number of its first entry there).
struct kv_view {
    const kv_seq * list;
    int32_t seqs;
    uint32_t * bad;
};

__device__ inline kv_seq load_seq(const kv_view & a, int b, int, bool &) { return a.list[b]; }

__device__ inline const int32_t * table_of(const kv_batch & a, const kv_seq & s) { return a.tables + (int64_t) s.slot * a.table_cols; }

// Where the sequences' runs of work lie: the sum of a cost over the sequences,
// and the sequence that holds a unit of it. Up to 64 sequences every wave keeps
// one a lane and finds them by a scan and a ballot, with no shared memory and no
// barrier (a call of few sequences is bound by such latencies); more go through
// prefix sums in shared memory (prefix[seqs + 1], whose barriers every thread of
// the workgroup reaches: threads a multiple of 64, at most 1024).
template <typename Cost, typename Batch> struct seq_index {
    const Batch & a;
    const int page_shift;
    int32_t * const prefix;
    kv_seq mine;
    int32_t incl, total;

    __device__ seq_index(const Batch & a, int page_shift, int32_t * prefix, Cost cost) : a(a), page_shift(page_shift), prefix(prefix) {
        const int lane = threadIdx.x & 63;
        bool bad = false;
        if (a.seqs <= 64) {
            mine = kv_seq{0, 0, 0, 0};
            if (lane < a.seqs) mine = load_seq(a, lane, page_shift, bad);
            incl = scan(lane < a.seqs ? cost(mine) : 0);
            total = __builtin_amdgcn_readlane(incl, 63);
        } else {
            __shared__ int32_t wave_sum[16];
            const int t = threadIdx.x, threads = blockDim.x;
            const int run = (a.seqs + threads - 1) / threads, first = min(t * run, a.seqs), last = min(first + run, a.seqs);
            int32_t sum = 0;
            for (int b = first; b < last; b++) {
                const int32_t c = cost(load_seq(a, b, page_shift, bad));
                prefix[b + 1] = c;
                sum = add(sum, c);
            }
            const int32_t s = scan(sum);
            if (lane == 63) wave_sum[t >> 6] = s;
            __syncthreads();
            const int32_t left = __shfl_up(s, 1);
            int32_t before = lane ? left : 0;
            for (int w = 0; w < (t >> 6); w++) before = add(before, wave_sum[w]);
            if (t == 0) prefix[0] = 0;
            for (int b = first; b < last; b++) prefix[b + 1] = before = add(before, prefix[b + 1]);
            __syncthreads();
            total = prefix[a.seqs];
        }
        if (bad && blockIdx.x == 0) report(a.bad);
    }

    // The units before sequence b, which need not be the same in every lane (every lane
    // calls it).
    __device__ int32_t before(int b) const {
        if (a.seqs > 64) return prefix[b];
        const int32_t upto = __shfl(incl, max(b - 1, 0));
        return b ? upto : 0;
    }

    // Sums stop at the type's limit: starts that go back make sequences overlap, and
    // their costs no longer keep to what the host bounds by the rows.
    static __device__ int32_t add(int32_t x, int32_t y) { return __builtin_elementwise_add_sat(x, y); }

    static __device__ int32_t scan(int32_t v) {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int32_t u = __shfl_up(v, off);
            if (lane >= off) v = add(v, u);
        }
        return v;
    }

    // The sequence that holds unit u < total (u and the answer the same in every
    // lane), and the units before it.
    __device__ kv_seq at(int32_t u, int32_t & before) const {
        if (a.seqs <= 64) {
            const int b = __popcll(__ballot(incl <= u));
            before = b ? __builtin_amdgcn_readlane(incl, max(b - 1, 0)) : 0;
            return kv_seq{__builtin_amdgcn_readlane(mine.row0, b), __builtin_amdgcn_readlane(mine.n, b),
                          __builtin_amdgcn_readlane(mine.len, b), __builtin_amdgcn_readlane(mine.slot, b)};
        }
        int lo = 0, hi = a.seqs;  // prefix[lo] <= u < prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= u) lo = mid;
            else hi = mid;
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        before = __builtin_amdgcn_readfirstlane(prefix[lo]);
        bool bad = false;
        return load_seq(a, lo, page_shift, bad);
    }
};

// Bytes of shared memory for seq_index's prefix sums.
inline size_t seq_index_bytes(int seqs) { return seqs <= 64 ? 0 : (size_t) ((seqs + 4) & ~3) * 4; }

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

// Whether two sets of rows (bytes apart, bytes long) share no byte: their spans lie
// apart, or they are column ranges of one wider buffer.
bool kv_rows_apart(const void * x, size_t ldx, size_t wx, const void * y, size_t ldy, size_t wy, int64_t rows);

// Bytes of a value of an F32, F16 or BF16 tensor, 0 for other types.
inline int kv_type_bytes(int type) {
    return type == ZEST_TYPE_F32 ? 4 : type == ZEST_TYPE_F16 || type == ZEST_TYPE_BF16 ? 2 : 0;
}

} // namespace zest

// The paged KV cache's upkeep: rope and the append into the pages, the
// scheduler's step over the page tables, compaction of the pool.
#include <algorithm>
#include <cmath>

#include "kv_device.h"
#include "zest_common.h"

namespace zest {

int kv_check_cache(const zest_kv_cache * c, const char * what) {
    ZEST_REQUIRE(c && c->pool, "%s: null cache", what);
    ZEST_REQUIRE(c->pages > 0 && c->pages <= (1 << 24), "%s: %lld pages (1 to 2^24)", what, (long long) c->pages);
    ZEST_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 1024, "%s: kv_heads=%d (1 to 1024)", what, c->kv_heads);
    const int d = c->head_dim, p = c->page_tokens;
    if (c->type != ZEST_TYPE_F16 && c->type != ZEST_TYPE_BF16)
        return fail(ZEST_E_UNSUPPORTED, "%s: cache type %d (F16 or BF16)", what, c->type);
    if (d != 64 && d != 96 && d != 128 && d != 192 && d != 256)
        return fail(ZEST_E_UNSUPPORTED, "%s: head_dim=%d (64, 96, 128, 192 or 256)", what, d);
    if (p != 16 && p != 32 && p != 64 && p != 128 && p != 256)
        return fail(ZEST_E_UNSUPPORTED, "%s: page_tokens=%d (16, 32, 64, 128 or 256)", what, p);
    ZEST_REQUIRE((reinterpret_cast<uintptr_t>(c->pool) & 15) == 0, "%s: the pool must be 16-byte aligned", what);
    return ZEST_OK;
}

int kv_check_batch(const zest_kv_cache * c, const zest_kv_batch * b, const char * what) {
    ZEST_REQUIRE(b && b->tables && b->lens && b->starts, "%s: null batch", what);
    ZEST_REQUIRE(b->seqs > 0 && b->seqs <= KV_MAX_SEQS, "%s: %d sequences (1 to %d)", what, b->seqs, KV_MAX_SEQS);
    ZEST_REQUIRE(b->rows > 0 && b->rows <= (1 << 27), "%s: %lld rows (1 to 2^27)", what, (long long) b->rows);
    ZEST_REQUIRE(b->table_rows > 0 && b->table_cols > 0 && (int64_t) b->table_cols * c->page_tokens < (1ll << 31),
                 "%s: page tables of %d x %d", what, b->table_rows, b->table_cols);
    ZEST_REQUIRE(b->slots || b->seqs <= b->table_rows, "%s: %d sequences of %d slots", what, b->seqs, b->table_rows);
    ZEST_REQUIRE(b->max_new > 0 && b->max_new <= b->rows && b->max_len >= 0 && b->max_len <= (1 << 30), "%s: max_new=%d max_len=%d of %lld rows", what,
                 b->max_new, b->max_len, (long long) b->rows);
    return ZEST_OK;
}

int kv_check_rows(int type, const void * p, int64_t ld, int64_t width, const char * what, const char * name) {
    const int size = kv_type_bytes(type);
    if (!size) return fail(ZEST_E_UNSUPPORTED, "%s: %s of type %d (F32, F16 or BF16)", what, name, type);
    ZEST_REQUIRE(p, "%s: null %s", what, name);
    ZEST_REQUIRE(ld >= width, "%s: %s rows of %lld values, %lld apart", what, name, (long long) width, (long long) ld);
    ZEST_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0, "%s: %s rows must be 16-byte aligned", what,
                 name);
    return ZEST_OK;
}

bool kv_rows_apart(const void * x, size_t ldx, size_t wx, const void * y, size_t ldy, size_t wy, int64_t rows) {
    const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), y0 = reinterpret_cast<uintptr_t>(y);
    const size_t last = (size_t) (rows - 1);
    if (x0 + last * ldx + wx <= y0 || y0 + last * ldy + wy <= x0) return true;
    if (last == 0 || ldx != ldy) return false;
    const size_t off = y0 >= x0 ? (y0 - x0) % ldx : (ldx - (x0 - y0) % ldx) % ldx;
    return off >= wx && off + wy <= ldx;
}

} // namespace zest

namespace {

using zest::kv_batch;
using zest::kv_pages;
using zest::kv_seq;

// ---- append ---------------------------------------------------------------------

// Eight values of a row of type TYPE (F32, F16 or BF16) at element offset e (a
// multiple of 8: whole 16-byte pieces), as floats; and one.
template <int TYPE> __device__ inline void load8(const void * p, int64_t e, float v[8]) {
    if constexpr (TYPE == ZEST_TYPE_F32) {
        const float4 a = *reinterpret_cast<const float4 *>((const float *) p + e);
        const float4 b = *reinterpret_cast<const float4 *>((const float *) p + e + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        return;
    }
    const uint4 q = *reinterpret_cast<const uint4 *>((const uint16_t *) p + e);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (TYPE == ZEST_TYPE_BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            v[2 * i] = (float) __builtin_bit_cast(_Float16, (uint16_t) w[i]);
            v[2 * i + 1] = (float) __builtin_bit_cast(_Float16, (uint16_t) (w[i] >> 16));
        }
    }
}

template <int TYPE> __device__ inline float load1(const void * p, int64_t e) {
    if constexpr (TYPE == ZEST_TYPE_F32) return ((const float *) p)[e];
    const uint16_t w = ((const uint16_t *) p)[e];
    return TYPE == ZEST_TYPE_BF16 ? __uint_as_float((uint32_t) w << 16) : (float) __builtin_bit_cast(_Float16, w);
}

// One value in a 16-bit type, rounded to nearest even.
__device__ inline uint16_t to16(float v, int type) {
    return type == ZEST_TYPE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16) v) : __builtin_bit_cast(uint16_t, (_Float16) v);
}

__device__ inline uint4 pack8(const float v[8], int type) {
    typedef float f32x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    const f32x8 x = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
    if (type == ZEST_TYPE_BF16) return __builtin_bit_cast(uint4, __builtin_convertvector(x, bf16x8));
    return __builtin_bit_cast(uint4, __builtin_convertvector(x, f16x8));
}

struct append_args {
    kv_pages c;
    kv_batch b;
    int32_t d, cache_type, q_out_type, q_heads, heads_each, q_parts, kv_parts;  // grid.y: q_parts, then kv_parts of k and of v
    const void * k, * v, * q;
    void * q_out;
    int64_t ldk, ldv, ldq, ldq_out;
    const double * freqs;  // null: no rope
    int32_t rot, neox;
    float magnitude;
    const int32_t * pos;
};

// How a token's head is dealt out as items, each one lane's, which reads all of
// an item before it writes any of it (q_out may be q): pieces of 8 values; with
// NeoX rope of whole pieces, two pieces that turn with each other (and what is
// behind the turned dims as pieces); with other NeoX rope, a pair or a value.
enum { ITEM_PIECE = 0, ITEM_PAIR = 1, ITEM_SINGLE = 2 };

// One workgroup takes the new tokens within 16 consecutive places of a sequence
// (the unit in which V is stored) and heads_each heads of q, k or v. Every thread
// requests its first BATCH items before the angles are made, once a workgroup in
// shared memory: position * frequency in 64 bits, reduced to a fraction of a turn
// there (rint and a subtraction: exact to 2^-53 of the turns), and sine and
// cosine of that in 32. HBM bound. K's lanes run over tokens first, so a piece
// row of 16 tokens is 256 contiguous bytes; V's over columns, 8 tokens a lane, so
// a wave reads whole rows and writes whole lines. 2048 tokens of 32 query and 8
// k/v heads of 128 from fp32: 21.5 us, 75 MB at 3.5 TB/s; a head at a time, its
// items on half of the threads, 32.5.
//
// BATCH 4, and 1 where no sequence has more than one new token: a quarter of the
// code, whose first fetch is a good part of so small a call (64 sequences of the
// Qwen3-4B shape 10.2 -> 5.1 us).
template <int IN, int MODE, int BATCH> __global__ __launch_bounds__(256) void append_kernel(append_args a) {
    constexpr int WIDTH = MODE == ITEM_PAIR ? 16 : MODE == ITEM_PIECE ? 8 : 2;
    extern __shared__ __align__(16) int32_t append_sh[];
    const int t = threadIdx.x, ps = a.c.page_shift, P = 1 << ps;
    const size_t prefix_words = a.b.seqs <= 64 ? 0 : (a.b.seqs + 4) & ~3;
    float2 * turn = reinterpret_cast<float2 *>(append_sh + prefix_words);  // [16][rot / 2]
    const zest::seq_index index(a.b, ps, append_sh, [](const kv_seq & s) { return s.n > 0 ? ((s.len - 1) >> 4) - ((s.len - s.n) >> 4) + 1 : 0; });
    if ((int32_t) blockIdx.x >= index.total) return;
    int32_t before;
    const kv_seq s = index.at((int32_t) blockIdx.x, before);
    const int32_t first = s.len - s.n;                                               // place of the first new token
    const int32_t p0 = ((first >> 4) + ((int32_t) blockIdx.x - before)) << 4;         // the 16 places
    const int32_t lo = max(p0, first), hi = min(p0 + 16, s.len);                     // of them, new
    const int32_t r0 = s.row0 + (lo - first);                                        // row of place lo
    const int n = hi - lo, D = a.d, half = a.rot / 2;

    // the page, looked at when the values requested after it are there
    const int32_t page = p0 >= 0 ? a.b.tables[(int64_t) s.slot * a.b.table_cols + (p0 >> ps)] : -1;
    auto there = [&]() { return (uint32_t) page < (uint32_t) a.c.pages; };
    auto page_at = [&]() { return reinterpret_cast<uint16_t *>(a.c.pool + (int64_t) page * a.c.page_bytes); };

    const bool is_q = (int) blockIdx.y < a.q_parts;
    const int part = is_q ? blockIdx.y : (blockIdx.y - a.q_parts) % a.kv_parts;
    const int head0 = part * a.heads_each, heads = min(a.heads_each, (is_q ? a.q_heads : a.c.kv_heads) - head0);

    if (!is_q && (int) blockIdx.y >= a.q_parts + a.kv_parts) {  // v: 8 tokens of a column a lane
        const int64_t unit_at = (int64_t) P * D + (int64_t) ((p0 & (P - 1)) >> 4) * 16 * D;
        if (n < 16) {  // not the whole unit: a value at a time
            for (uint32_t x = t; x < (uint32_t) (heads * n * D); x += 256) {
                const uint32_t rest = x / D, e = x - rest * D, head = rest / n, tok = rest - head * n, at = lo + tok - p0;
                const float v = load1<IN>(a.v, (int64_t) (r0 + tok) * a.ldv + (int64_t) (head0 + head) * D + e);
                if (there())
                    page_at()[unit_at + (int64_t) (head0 + head) * 2 * P * D + ((at >> 2 & 1) * D + e) * 8 + (at & 3) + (at >> 3) * 4] =
                        to16(v, a.cache_type);
            }
            if (!there() && t == 0) zest::report(a.b.bad);
            return;
        }
        const uint32_t total = heads * 2 * D, per = 2 * D;
        for (uint32_t base = t; base < total; base += 256 * BATCH) {
            float o[BATCH][8];
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                const uint32_t x = base + 256 * u, head = head0 + x / per, i = x % per;
                const int h = i >= (uint32_t) D, e = i - h * D;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int tok = 4 * h + (j & 3) + (j >> 2) * 8;
                    o[u][j] = x < total ? load1<IN>(a.v, (int64_t) (r0 + tok) * a.ldv + (int64_t) head * D + e) : 0.0f;
                }
            }
            if (!there()) {
                if (t == 0) zest::report(a.b.bad);
                return;
            }
#pragma unroll
            for (int u = 0; u < BATCH; u++) {
                const uint32_t x = base + 256 * u, head = head0 + x / per, i = x % per;
                if (x >= total) break;
                *reinterpret_cast<uint4 *>(page_at() + unit_at + (int64_t) head * 2 * P * D + i * 8) = pack8(o[u], a.cache_type);
            }
        }
        return;
    }

    const uint32_t turning = MODE == ITEM_PAIR ? half / 8 : MODE == ITEM_SINGLE ? half : 0;
    const uint32_t items = MODE == ITEM_SINGLE ? half + (D - a.rot) : MODE == ITEM_PAIR ? half / 8 + (D - a.rot) / 8 : D / 8;
    const uint32_t total = heads * n * items;
    const void * const src = is_q ? a.q : a.k;
    const int64_t ld = is_q ? a.ldq : a.ldk;
    // item x: q's lanes over a token's items first, k's over the tokens
    auto place_of = [&](uint32_t x, uint32_t & head, uint32_t & i) {
        const uint32_t inner = is_q ? items : n, rest = x / inner, fast = x - rest * inner, outer = is_q ? n : items;
        head = rest / outer;
        const uint32_t slow = rest - head * outer;
        head += head0;
        i = is_q ? fast : slow;
        return x < total ? (int) (is_q ? slow : fast) : -1;
    };
    for (uint32_t base = 0; base < total || base == 0; base += 256 * BATCH) {
        float o[BATCH][WIDTH];
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            uint32_t head, i;
            const int tok = place_of(base + t + 256 * u, head, i);
            if (tok < 0) continue;
            const int64_t at = (r0 + tok) * ld + (int64_t) head * D;
            if constexpr (MODE == ITEM_SINGLE) {
                o[u][0] = load1<IN>(src, i < turning ? at + i : at + i + half);
                if (i < turning) o[u][1] = load1<IN>(src, at + i + half);
            } else if constexpr (MODE == ITEM_PAIR) {
                load8<IN>(src, i < turning ? at + 8 * i : at + a.rot + 8 * (i - turning), o[u]);
                if (i < turning) load8<IN>(src, at + 8 * i + half, o[u] + 8);
            } else {
                load8<IN>(src, at + 8 * i, o[u]);
            }
        }
        if (base == 0 && a.freqs) {
            for (int i = t; i < n * half; i += 256) {
                const int tok = i / half, p = i - tok * half;
                const double x = (double) (a.pos ? a.pos[r0 + tok] : lo + tok) * a.freqs[p] * 0.15915494309189535;  // turns
                const float f = (float) (x - rint(x));
                float sn, cs;
                sincospif(2.0f * f, &sn, &cs);
                turn[i] = make_float2(cs * a.magnitude, sn * a.magnitude);
            }
            __syncthreads();
        }
        if (!is_q && !there()) return;  // v's workgroup reports it
        uint16_t * const held = is_q ? nullptr : page_at();
#pragma unroll
        for (int u = 0; u < BATCH; u++) {
            uint32_t head, i;
            const int tok = place_of(base + t + 256 * u, head, i);
            if (tok < 0) continue;
            const int64_t row = (r0 + tok) * a.ldq_out + (int64_t) head * D;
            uint16_t * y = held + (int64_t) head * 2 * P * D + ((lo + tok) & (P - 1)) * 8;  // k: its token's first piece
            auto put8 = [&](int e, const float * v) {
                if (!is_q) {
                    *reinterpret_cast<uint4 *>(y + (int64_t) e * P) = pack8(v, a.cache_type);
                } else if (a.q_out_type == ZEST_TYPE_F32) {
                    float * z = (float *) a.q_out + row + e;
                    *reinterpret_cast<float4 *>(z) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4 *>(z + 4) = make_float4(v[4], v[5], v[6], v[7]);
                } else {
                    *reinterpret_cast<uint4 *>((uint16_t *) a.q_out + row + e) = pack8(v, a.q_out_type);
                }
            };
            auto put1 = [&](int e, float v) {
                if (!is_q) y[(int64_t) (e / 8) * P * 8 + e % 8] = to16(v, a.cache_type);
                else if (a.q_out_type == ZEST_TYPE_F32) ((float *) a.q_out)[row + e] = v;
                else ((uint16_t *) a.q_out)[row + e] = to16(v, a.q_out_type);
            };
            const float2 * cs = turn + tok * half;
            if constexpr (MODE == ITEM_SINGLE) {
                if (i < turning) {
                    const float2 r = cs[i];
                    put1(i, fmaf(o[u][0], r.x, -(o[u][1] * r.y)));
                    put1(i + half, fmaf(o[u][0], r.y, o[u][1] * r.x));
                } else {
                    put1(i + half, o[u][0]);
                }
            } else if constexpr (MODE == ITEM_PAIR) {
                if (i < turning) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float2 r = cs[8 * i + j];
                        const float x0 = o[u][j], x1 = o[u][8 + j];
                        o[u][j] = fmaf(x0, r.x, -(x1 * r.y));
                        o[u][8 + j] = fmaf(x0, r.y, x1 * r.x);
                    }
                    put8(8 * i, o[u]);
                    put8(8 * i + half, o[u] + 8);
                } else {
                    put8(a.rot + 8 * (i - turning), o[u]);
                }
            } else {
                if (a.freqs) {
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        if (8 * i + j < (uint32_t) a.rot) {
                            const float2 r = cs[4 * i + j / 2];
                            const float x0 = o[u][j], x1 = o[u][j + 1];
                            o[u][j] = fmaf(x0, r.x, -(x1 * r.y));
                            o[u][j + 1] = fmaf(x0, r.y, x1 * r.x);
                        }
                    }
                }
                put8(8 * i, o[u]);
            }
        }
    }
}

// ---- the scheduler's step --------------------------------------------------------

constexpr int MAX_SLOTS = 65536, MAX_ENTRIES = 65536;
constexpr int STEP = 1024;  // threads of the one workgroup that walks the tables

// A count that other threads of this workgroup changed with atomics: read past
// the vector cache.
__device__ inline int32_t fresh(const int32_t * p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// Exclusive scan of one value a thread (0 to MOST) over a 1024-thread workgroup;
// *total its sum. Sums stop at MOST, more than any pool has pages, so that no
// list of wishes wraps around. Ends in a barrier.
constexpr int32_t MOST = 1 << 29;

__device__ inline int32_t scan_step(int32_t v, int32_t * total) {
    __shared__ int32_t sums[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t u = __shfl_up(s, off);
        if (lane >= off) s = min(s + u, MOST);
    }
    if (lane == 63) sums[wave] = s;
    __syncthreads();
    int32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        before = min(before + (w < wave ? sums[w] : 0), MOST);
        all = min(all + sums[w], MOST);
    }
    __syncthreads();
    *total = all;
    const int32_t left = __shfl_up(s, 1);
    return min(before + (lane ? left : 0), MOST);
}

// An entry between the phases of assign_kernel (base -1: left undone).
struct assign_entry {
    int32_t base, need, first, old_pages;
};

struct assign_args {
    int32_t * refs, * tables, * lens;
    const int32_t * dst, * src, * grow;
    int32_t n, rows, cols, pages, page_shift;
    assign_entry * entries;  // [n]
    int2 * copies;           // [n]: the page a fork's open page is copied from, and to (-1: none)
    int32_t * free_list;     // [pages]
    uint32_t * bad;
};

// Working memory of the one-workgroup kernels below that fits shared memory: a
// round trip to global memory between phases costs more than the phase.
constexpr int FEW_ENTRIES = 512, FEW_PAGES = 4096;

// The tables' part of a step, by one workgroup: its phases are ordered by
// barriers, so every count is exact and the result does not depend on the order
// of the atomics (sums only). Latency bound: a chain of a few dependent accesses
// (12 slots of up to 13 pages: 8.2 to 9.0 us, with entries and free pages in global memory
// 12.3).
__global__ __launch_bounds__(STEP) void assign_kernel(assign_args a) {
    __shared__ uint32_t seen[MAX_SLOTS / 32], twice[MAX_SLOTS / 32], replaced[MAX_SLOTS / 32];
    __shared__ assign_entry few_entries[FEW_ENTRIES];
    __shared__ int32_t few_pages[FEW_PAGES];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int P = 1 << a.page_shift;
    assign_entry * const entries = a.n <= FEW_ENTRIES ? few_entries : a.entries;
    int32_t * const free_list = a.pages <= FEW_PAGES ? few_pages : a.free_list;
    bool bad = false;
    for (int i = t; i < (a.rows + 31) / 32; i += STEP) seen[i] = twice[i] = replaced[i] = 0;
    __syncthreads();
    for (int i = t; i < a.n; i += STEP) {
        const int32_t d = a.dst[i], s = a.src[i];
        if ((uint32_t) d >= (uint32_t) a.rows) continue;
        const uint32_t bit = 1u << (d & 31);
        if (atomicOr(&seen[d >> 5], bit) & bit) atomicOr(&twice[d >> 5], bit);
        if (s != d) atomicOr(&replaced[d >> 5], bit);
    }
    __syncthreads();
    auto has = [](const uint32_t * set, int32_t d) { return (set[d >> 5] >> (d & 31)) & 1u; };

    // what each entry needs, and its place in the list of free pages
    int32_t want = 0;
    for (int i0 = 0; i0 < a.n; i0 += STEP) {
        const int i = i0 + t;
        assign_entry e{-1, 0, 0, 0};
        if (i < a.n) {
            const int32_t d = a.dst[i], s = a.src[i], g = a.grow[i];
            const bool named = (uint32_t) d < (uint32_t) a.rows && s >= -1 && s < a.rows;
            const int32_t held_base = a.lens[named && s >= 0 ? s : 0], held_old = a.lens[named ? d : 0];
            if (named && !has(twice, d) && (s < 0 || s == d || !has(replaced, s)) && g >= 0) {
                const int64_t base = s >= 0 ? held_base : 0, room = (int64_t) a.cols << a.page_shift, old = held_old;
                if (base >= 0 && base + g <= room && old >= 0 && old <= room) {
                    e.base = (int32_t) base;
                    const int32_t held = (int32_t) (s == d ? (base + P - 1) >> a.page_shift : base >> a.page_shift);
                    e.need = min((int32_t) ((base + g + P - 1) >> a.page_shift) - held, MOST);
                    e.old_pages = s == d ? 0 : (int32_t) ((old + P - 1) >> a.page_shift);
                }
            }
            bad |= e.base < 0;
        }
        int32_t sum;
        e.first = min(want + scan_step(e.need, &sum), MOST);
        want = min(want + sum, MOST);
        if (i < a.n) {
            entries[i] = e;
            a.copies[i] = make_int2(-1, -1);
        }
    }
    __syncthreads();

    // the replaced rows' pages are released, a wave an entry
    for (int i = wave; i < a.n; i += STEP / 64) {
        const assign_entry e = entries[i];
        if (e.base < 0 || e.old_pages == 0) continue;
        const int32_t * row = a.tables + (int64_t) a.dst[i] * a.cols;
        for (int j = lane; j < e.old_pages; j += 64) {
            const int32_t id = row[j];
            if (id == -1) continue;  // a window has left it
            if ((uint32_t) id >= (uint32_t) a.pages) bad = true;
            else if (atomicSub(&a.refs[id], 1) <= 0) {  // not counted: left at what it was
                atomicAdd(&a.refs[id], 1);
                bad = true;
            }
        }
    }
    __threadfence();
    __syncthreads();

    int32_t found = 0;
    for (int p0 = 0; p0 < a.pages && found < want; p0 += STEP) {
        const int p = p0 + t;
        const bool is_free = p < a.pages && fresh(&a.refs[p]) <= 0;
        int32_t sum;
        const int32_t before = scan_step(is_free, &sum);
        if (is_free && found + before < want) free_list[found + before] = p;
        found += sum;
    }
    __syncthreads();

    // the new rows, a wave an entry
    for (int i = wave; i < a.n; i += STEP / 64) {
        const assign_entry e = entries[i];
        if (e.base < 0) continue;
        const int32_t d = a.dst[i], s = a.src[i], g = a.grow[i];
        int32_t * row = a.tables + (int64_t) d * a.cols;
        const bool fits = e.need == 0 || e.first + e.need <= found;
        bad |= !fits;
        if (s == d) {
            if (!fits) continue;
            const int32_t held = (e.base + P - 1) >> a.page_shift;
            for (int j = lane; j < e.need; j += 64) {
                const int32_t id = free_list[e.first + j];
                row[held + j] = id;
                a.refs[id] = 1;
            }
            if (lane == 0) a.lens[d] = e.base + g;
            continue;
        }
        const int32_t * parent = a.tables + (int64_t) max(s, 0) * a.cols;
        const int32_t shared = fits ? e.base >> a.page_shift : 0, total = fits ? shared + e.need : 0;
        for (int j = lane; j < a.cols; j += 64) {
            int32_t id = -1;
            if (j < shared) {
                id = parent[j];
                if ((uint32_t) id < (uint32_t) a.pages) atomicAdd(&a.refs[id], 1);
                else bad |= id != -1;
            } else if (j < total) {
                id = free_list[e.first + j - shared];
                a.refs[id] = 1;
                if (j == shared && (e.base & (P - 1))) {
                    const int32_t from = parent[j];
                    if ((uint32_t) from < (uint32_t) a.pages) a.copies[i] = make_int2(from, id);
                    else bad = true;
                }
            }
            row[j] = id;
        }
        if (lane == 0) a.lens[d] = fits ? e.base + g : 0;
    }
    if (bad) zest::report(a.bad);
}

// Copies n whole pages in every layer, copies[i] = (from, to), -1 for none; by
// `blocks` workgroups of 256 threads, each COPY_BYTES of a page at a time, four
// 16-byte loads a thread before the first store. Memory bound: 40 forks' open pages
// in 36 layers, 755 MB, 113 us, and 3.4 GB in 680 us, at a copy's rate.
constexpr int COPY_BYTES = 16384;

__device__ inline void copy_pages(uint8_t * pool, int64_t page_bytes, int64_t layer_stride, int32_t layers, const int2 * copies,
                                  int32_t n, int32_t block, int32_t blocks) {
    const int32_t parts = (int32_t) ((page_bytes + COPY_BYTES - 1) / COPY_BYTES);
    const int64_t total = (int64_t) n * layers * parts;
    for (int64_t w = block; w < total; w += blocks) {
        const int32_t part = (int32_t) (w % parts), layer = (int32_t) (w / parts % layers);
        const int2 c = copies[w / parts / layers];
        if (c.x < 0) continue;
        const int64_t at = layer * layer_stride + (int64_t) part * COPY_BYTES;
        const int32_t left = (int32_t) min((int64_t) COPY_BYTES, page_bytes - (int64_t) part * COPY_BYTES);
        const uint4 * from = reinterpret_cast<const uint4 *>(pool + at + c.x * page_bytes);
        uint4 * to = reinterpret_cast<uint4 *>(pool + at + c.y * page_bytes);
        const int t = threadIdx.x, last = left / 16 - 1;  // the part's end is read again rather than past it
        const uint4 v0 = from[min(t, last)], v1 = from[min(t + 256, last)];
        const uint4 v2 = from[min(t + 512, last)], v3 = from[min(t + 768, last)];
        if (t <= last) to[t] = v0;
        if (t + 256 <= last) to[t + 256] = v1;
        if (t + 512 <= last) to[t + 512] = v2;
        if (t + 768 <= last) to[t + 768] = v3;
    }
}

__global__ __launch_bounds__(256) void copy_pages_kernel(uint8_t * pool, int64_t page_bytes, int64_t layer_stride, int32_t layers,
                                                         const int2 * copies, int32_t n) {
    copy_pages(pool, page_bytes, layer_stride, layers, copies, n, blockIdx.x, gridDim.x);
}

// ---- compaction ------------------------------------------------------------------

struct compact_args {
    const int32_t * refs, * tables;
    int32_t * refs_out, * tables_out, * live;
    int32_t pages;
    int64_t entries;
    int2 * moves;       // [pages / 2 + 1]: from, to
    int32_t * count;    // of them
    int32_t * place;    // [pages]: where a page is afterwards, -1 for one without references
    uint32_t * bad;
};

// Which page moves where, by one workgroup: a count of the live pages, then the
// free pages below it and the live ones from it on, which are equally many: rank k
// of these goes to rank k of those.
__global__ __launch_bounds__(STEP) void compact_plan_kernel(compact_args a) {
    __shared__ int32_t few_holes[FEW_PAGES];
    const int t = threadIdx.x;
    int32_t mine = 0, live;
    for (int p = t; p < a.pages; p += STEP) mine += a.refs[p] > 0;
    scan_step(mine, &live);
    const bool few = live <= FEW_PAGES;
    int32_t holes = 0;
    for (int p0 = 0; p0 < live; p0 += STEP) {
        const int p = p0 + t;
        const int32_t refs = p < live ? a.refs[p] : 1;
        int32_t sum;
        const int32_t before = holes + scan_step(refs <= 0, &sum);
        if (refs <= 0) {
            if (few) few_holes[before] = p;
            else a.moves[before].y = p;
        }
        if (p < live) {
            a.place[p] = refs > 0 ? p : -1;
            if (refs > 0) a.refs_out[p] = refs;
        }
        holes += sum;
    }
    __syncthreads();
    int32_t movers = 0;
    for (int p0 = live; p0 < a.pages; p0 += STEP) {
        const int p = p0 + t;
        const int32_t refs = p < a.pages ? a.refs[p] : 0;
        int32_t sum;
        const int32_t k = movers + scan_step(refs > 0, &sum);
        if (refs > 0) {
            const int32_t to = few ? few_holes[k] : a.moves[k].y;
            a.moves[k] = make_int2(p, to);
            a.place[p] = to;
            a.refs_out[to] = refs;
        } else if (p < a.pages) {
            a.place[p] = -1;
        }
        if (p < a.pages) a.refs_out[p] = 0;  // refs_out may be refs: this page's count has been read
        movers += sum;
    }
    if (t == 0) {
        *a.count = movers;
        *a.live = live;
    }
}

// The tables, by the first table_blocks workgroups, and beside them the pages.
__global__ __launch_bounds__(256) void compact_move_kernel(compact_args a, int32_t table_blocks, uint8_t * pool, int64_t page_bytes,
                                                           int64_t layer_stride, int32_t layers) {
    if ((int32_t) blockIdx.x >= table_blocks) {
        copy_pages(pool, page_bytes, layer_stride, layers, a.moves, *a.count, blockIdx.x - table_blocks, gridDim.x - table_blocks);
        return;
    }
    bool bad = false;
    for (int64_t i = (int64_t) blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t) table_blocks * 256) {
        const int32_t id = a.tables[i];
        const int32_t to = (uint32_t) id < (uint32_t) a.pages ? a.place[id] : -1;
        bad |= to < 0 && id != -1;
        a.tables_out[i] = to;
    }
    if (bad) zest::report(a.bad);
}

size_t round16(size_t n) { return (n + 15) & ~(size_t) 15; }

int check_pool(const zest_kv_cache * c, int32_t layers, int64_t layer_stride, const int32_t * refs, const int32_t * tables,
               int32_t table_rows, int32_t table_cols, const char * what) {
    if (const int st = zest::kv_check_cache(c, what)) return st;
    ZEST_REQUIRE(layers > 0 && layers <= 65536, "%s: %d layers", what, layers);
    ZEST_REQUIRE(layers == 1 || (layer_stride % 16 == 0 && layer_stride >= c->pages * (int64_t) zest_kv_page_bytes(c)),
                 "%s: layers %lld bytes apart", what, (long long) layer_stride);
    ZEST_REQUIRE(refs && tables, "%s: null refs or tables", what);
    ZEST_REQUIRE(table_rows > 0 && table_rows <= MAX_SLOTS && table_cols > 0 &&
                     (int64_t) table_cols * c->page_tokens < (1ll << 31),
                 "%s: page tables of %d x %d", what, table_rows, table_cols);
    return ZEST_OK;
}

unsigned copy_grid(const zest_kv_cache * c, int32_t layers, int64_t n) {
    const int64_t parts = ((int64_t) zest_kv_page_bytes(c) + COPY_BYTES - 1) / COPY_BYTES;
    return (unsigned) std::min<int64_t>(n * layers * parts, 8192);
}

} // namespace

extern "C" {

size_t zest_kv_page_bytes(const zest_kv_cache * c) {
    return c ? (size_t) c->kv_heads * 4 * (size_t) c->page_tokens * (size_t) c->head_dim : 0;
}

int zest_kv_rope_freqs(int32_t n_dims, double freq_base, double freq_scale, double ext_factor, double attn_factor,
                       double corr0, double corr1, const float * ff, double * out, float * magnitude) {
    ZEST_REQUIRE(out && magnitude, "zest_kv_rope_freqs: null pointer");
    ZEST_REQUIRE(n_dims > 0 && n_dims % 2 == 0, "zest_kv_rope_freqs: n_dims=%d", n_dims);
    ZEST_REQUIRE(freq_base > 0 && freq_scale > 0, "zest_kv_rope_freqs: base %g, scale %g", freq_base, freq_scale);
    for (int p = 0; p < n_dims / 2; p++) {
        const double f = std::pow(freq_base, -2.0 * p / n_dims) / (ff ? (double) ff[p] : 1.0);
        const double y = (p - corr0) / std::max(0.001, corr1 - corr0);
        const double mix = (1.0 - std::min(1.0, std::max(0.0, y))) * ext_factor;
        out[p] = f * (freq_scale * (1.0 - mix) + mix);
    }
    *magnitude = (float) (attn_factor * (ext_factor != 0.0 ? 1.0 + 0.1 * std::log(1.0 / freq_scale) : 1.0));
    return ZEST_OK;
}

int zest_kv_append(const zest_kv_cache * cache, const zest_kv_batch * batch, const zest_kv_rope * rope, const int32_t * pos,
                   int in_type, const void * k, int64_t ldk, const void * v, int64_t ldv, const void * q, int64_t ldq,
                   int32_t q_heads, void * q_out, int64_t ldq_out, int q_out_type, uint32_t * bad, void * stream) {
    const char * me = "zest_kv_append";
    if (const int st = zest::kv_check_cache(cache, me)) return st;
    if (const int st = zest::kv_check_batch(cache, batch, me)) return st;
    const int64_t width = (int64_t) cache->kv_heads * cache->head_dim;
    if (const int st = zest::kv_check_rows(in_type, k, ldk, width, me, "k")) return st;
    if (const int st = zest::kv_check_rows(in_type, v, ldv, width, me, "v")) return st;
    if (q) {
        ZEST_REQUIRE(q_heads > 0 && q_heads <= 4096, "%s: q_heads=%d (1 to 4096)", me, q_heads);
        if (const int st = zest::kv_check_rows(in_type, q, ldq, (int64_t) q_heads * cache->head_dim, me, "q")) return st;
        if (const int st = zest::kv_check_rows(q_out_type, q_out, ldq_out, (int64_t) q_heads * cache->head_dim, me, "q_out"))
            return st;
        // q, k and v are different workgroups' work, in no order
        const size_t is = zest::kv_type_bytes(in_type), os = zest::kv_type_bytes(q_out_type), row = (size_t) q_heads * cache->head_dim;
        auto apart = [&](const void * x, int64_t ld, size_t w) {
            return zest::kv_rows_apart(x, ld * is, w * is, q_out, ldq_out * os, row * os, batch->rows);
        };
        ZEST_REQUIRE((q == q_out && ldq == ldq_out && in_type == q_out_type) || apart(q, ldq, row), "%s: q_out overlaps q without being q",
                     me);
        ZEST_REQUIRE(apart(k, ldk, width) && apart(v, ldv, width), "%s: q_out overlaps k or v", me);
        ZEST_REQUIRE(zest::kv_rows_apart(cache->pool, 0, cache->pages * zest_kv_page_bytes(cache), q_out, 0,
                                         ((batch->rows - 1) * ldq_out + row) * os, 1),
                     "%s: q_out overlaps the pool", me);
    }
    if (rope) {
        ZEST_REQUIRE(rope->freqs && (reinterpret_cast<uintptr_t>(rope->freqs) & 7) == 0, "%s: null or misaligned freqs", me);
        ZEST_REQUIRE(rope->n_dims > 0 && rope->n_dims % 2 == 0 && rope->n_dims <= cache->head_dim, "%s: n_dims=%d of %d", me,
                     rope->n_dims, cache->head_dim);
        ZEST_REQUIRE(rope->mode == 0 || rope->mode == 2, "%s: rope mode %d (normal 0 or neox 2)", me, rope->mode);
    }
    append_args a{};
    a.c = zest::kv_pages_of(cache);
    a.b = zest::kv_batch_of(batch, bad);
    a.d = cache->head_dim;
    a.cache_type = cache->type;
    a.q_out_type = q_out_type;
    a.q_heads = q ? q_heads : 0;
    a.k = k, a.v = v, a.q = q, a.q_out = q_out;
    a.ldk = ldk, a.ldv = ldv, a.ldq = ldq, a.ldq_out = ldq_out;
    if (rope) {
        a.freqs = rope->freqs;
        a.rot = rope->n_dims;
        a.neox = rope->mode == 2;
        a.magnitude = rope->magnitude;
    }
    a.pos = pos;
    // n new tokens of a sequence touch at most n / 16 + 2 units of 16 places, and at most n
    const int64_t units = std::min<int64_t>(batch->rows, batch->rows / 16 + 2ll * batch->seqs);
    const int heads = a.q_heads + 2 * a.c.kv_heads;
    // eight heads a workgroup (four items a thread of a 128-wide NeoX head), fewer
    // where that would leave CUs without one
    a.heads_each = (int) std::max<int64_t>(1, std::min<int64_t>(8, units * heads / 512));
    a.q_parts = (a.q_heads + a.heads_each - 1) / a.heads_each;
    a.kv_parts = (a.c.kv_heads + a.heads_each - 1) / a.heads_each;
    const size_t lds = zest::seq_index_bytes(batch->seqs) + (size_t) 16 * (a.rot / 2) * sizeof(float2);
    const dim3 grid((unsigned) units, (unsigned) (a.q_parts + 2 * a.kv_parts));
    const int mode = !a.neox ? ITEM_PIECE : a.rot % 16 == 0 ? ITEM_PAIR : ITEM_SINGLE;
    const bool one = batch->max_new == 1;
    const hipStream_t s = zest::as_stream(stream);
#define ZEST_APPEND(IN)                                                                                              \
    hipLaunchKernelGGL((mode == ITEM_PIECE  ? (one ? append_kernel<IN, ITEM_PIECE, 1> : append_kernel<IN, ITEM_PIECE, 4>) \
                        : mode == ITEM_PAIR ? (one ? append_kernel<IN, ITEM_PAIR, 1> : append_kernel<IN, ITEM_PAIR, 4>)   \
                                            : append_kernel<IN, ITEM_SINGLE, 4>),                                         \
                       grid, dim3(256), lds, s, a)
    if (in_type == ZEST_TYPE_F32) ZEST_APPEND(ZEST_TYPE_F32);
    else if (in_type == ZEST_TYPE_BF16) ZEST_APPEND(ZEST_TYPE_BF16);
    else ZEST_APPEND(ZEST_TYPE_F16);
#undef ZEST_APPEND
    return zest::check_launch(me);
}

size_t zest_kv_scratch_bytes(int64_t pages, int32_t n) {
    if (pages <= 0 || n < 0) return 0;
    const size_t assign = round16((size_t) n * sizeof(assign_entry)) + round16((size_t) n * sizeof(int2)) + round16((size_t) pages * 4);
    const size_t compact = round16((size_t) (pages / 2 + 1) * sizeof(int2)) + 16 + round16((size_t) pages * 4);
    return std::max(assign, compact);
}

int zest_kv_assign(const zest_kv_cache * cache, int32_t layers, int64_t layer_stride, int32_t * refs, int32_t * tables,
                   int32_t * lens, int32_t table_rows, int32_t table_cols, const int32_t * dst, const int32_t * src,
                   const int32_t * grow, int32_t n, void * scratch, size_t scratch_bytes, uint32_t * bad, void * stream) {
    const char * me = "zest_kv_assign";
    if (const int st = check_pool(cache, layers, layer_stride, refs, tables, table_rows, table_cols, me)) return st;
    ZEST_REQUIRE(lens && dst && src && grow, "%s: null pointer", me);
    ZEST_REQUIRE(n > 0 && n <= MAX_ENTRIES, "%s: %d entries (1 to %d)", me, n, MAX_ENTRIES);
    ZEST_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 &&
                     scratch_bytes >= zest_kv_scratch_bytes(cache->pages, n),
                 "%s: scratch of %zu bytes, 16-byte aligned, wanted", me, zest_kv_scratch_bytes(cache->pages, n));
    assign_args a{};
    a.refs = refs, a.tables = tables, a.lens = lens;
    a.dst = dst, a.src = src, a.grow = grow;
    a.n = n, a.rows = table_rows, a.cols = table_cols, a.pages = (int32_t) cache->pages;
    a.page_shift = zest::kv_page_shift(cache->page_tokens);
    uint8_t * at = (uint8_t *) scratch;
    a.entries = (assign_entry *) at;
    at += round16((size_t) n * sizeof(assign_entry));
    a.copies = (int2 *) at;
    at += round16((size_t) n * sizeof(int2));
    a.free_list = (int32_t *) at;
    a.bad = bad;
    const hipStream_t s = zest::as_stream(stream);
    hipLaunchKernelGGL(assign_kernel, dim3(1), dim3(STEP), 0, s, a);
    if (const int st = zest::check_launch(me)) return st;
    hipLaunchKernelGGL(copy_pages_kernel, dim3(copy_grid(cache, layers, n)), dim3(256), 0, s, (uint8_t *) cache->pool,
                       (int64_t) zest_kv_page_bytes(cache), layer_stride, layers, a.copies, n);
    return zest::check_launch(me);
}

int zest_kv_compact(const zest_kv_cache * cache, int32_t layers, int64_t layer_stride, const int32_t * refs,
                    const int32_t * tables, int32_t table_rows, int32_t table_cols, int32_t * refs_out, int32_t * tables_out,
                    int32_t * live, void * scratch, size_t scratch_bytes, uint32_t * bad, void * stream) {
    const char * me = "zest_kv_compact";
    if (const int st = check_pool(cache, layers, layer_stride, refs, tables, table_rows, table_cols, me)) return st;
    ZEST_REQUIRE(refs_out && tables_out && live, "%s: null pointer", me);
    ZEST_REQUIRE(scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 &&
                     scratch_bytes >= zest_kv_scratch_bytes(cache->pages, 0),
                 "%s: scratch of %zu bytes, 16-byte aligned, wanted", me, zest_kv_scratch_bytes(cache->pages, 0));
    compact_args a{};
    a.refs = refs, a.tables = tables, a.refs_out = refs_out, a.tables_out = tables_out, a.live = live;
    a.pages = (int32_t) cache->pages;
    a.entries = (int64_t) table_rows * table_cols;
    uint8_t * at = (uint8_t *) scratch;
    a.moves = (int2 *) at;
    at += round16((size_t) (cache->pages / 2 + 1) * sizeof(int2));
    a.count = (int32_t *) at;
    a.place = (int32_t *) (at + 16);
    a.bad = bad;
    const hipStream_t s = zest::as_stream(stream);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(STEP), 0, s, a);
    if (const int st = zest::check_launch(me)) return st;
    const int32_t table_blocks = (int32_t) std::min<int64_t>((a.entries + 255) / 256, 1024);
    hipLaunchKernelGGL(compact_move_kernel, dim3(table_blocks + copy_grid(cache, layers, cache->pages / 2 + 1)), dim3(256), 0, s, a,
                       table_blocks, (uint8_t *) cache->pool, (int64_t) zest_kv_page_bytes(cache), layer_stride, layers);
    return zest::check_launch(me);
}

} // extern "C"

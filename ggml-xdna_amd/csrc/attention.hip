// Attention over the paged KV cache (include/zest/kv.h): one pass over the keys
// with the running maximum and sum of a softmax, on v_mfma_f32_32x32x16 (many
// columns) or 16x16x32 (few).
//
// A column is one (new token, query head) pair of a k/v head, token-major: with
// a group of G query heads column c is token c / G and head c % G of the group,
// so one token's heads share the keys and values that a wave reads, and a chunk
// of tokens fills whole tiles. Scores are computed as S^T = K Q^T: 32 tokens by
// 32 columns, K the A operand and Q^T, held in registers, the B operand. A lane
// then holds 16 scores of one column (column lane % 32; tokens 8k + 4h + 0..3
// for k = 0..3, h = lane / 32), so the softmax statistics are one value a lane
// and need one exchange between lane halves a tile. O^T = V^T P^T takes the
// weights as its B operand from the registers they are in: the contraction runs
// over tokens in the order 4h..4h+3, 8+4h..8+4h+3 of each 16, which is the order
// the cache stores V in.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "kv_device.h"
#include "zest_common.h"

namespace {

using zest::kv_batch;
using zest::kv_pages;
using zest::kv_seq;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr int WAVES = 4;     // waves of a workgroup
constexpr int GROUP = 32;    // tokens a wave takes at a time
constexpr int UNIT = WAVES * GROUP;  // tokens of a unit of work
constexpr int CUS = 256;
// The most columns of a sequence that attend_few takes: two of its tiles, each of
// which reads K and V, where all that a call's bounds let it read stays in the
// 256 MB last-level cache (9 short sequences of the small model 20.6 us, with one
// tile 25.4), else one (16 sequences of 12 drafted tokens, 48 columns, at 4096 to
// 8192 tokens 105.7 us, with two tiles 126.2).
constexpr int most_few_cols(double kv_bytes) { return kv_bytes <= 256e6 ? 64 : 32; }

// The cache's element type: its fragment, its MFMA and its exponent field.
template <int TYPE> struct elem;

template <> struct elem<ZEST_TYPE_BF16> {
    typedef bf16x8 frag;
    static constexpr uint32_t EXP = 0x7f807f80u, ONE = 0x00800080u;
    // exponent added to the softmax weights: none, bf16 has fp32's range
    static constexpr float SHIFT = 0.0f;
    static __device__ f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mfma16(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __bf16 from(float v) { return (__bf16) v; }
};

template <> struct elem<ZEST_TYPE_F16> {
    typedef f16x8 frag;
    static constexpr uint32_t EXP = 0x7c007c00u, ONE = 0x04000400u;
    // weights are held times 2^6 (the sum with them, so it cancels): one 2^-20 of
    // the largest is still a normal fp16 number, and 2^(6 + SLACK) is in range
    static constexpr float SHIFT = 6.0f;
    static __device__ f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    static __device__ f32x4 mfma16(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ _Float16 from(float v) { return (_Float16) v; }
};

struct attn_args {
    kv_pages c;
    kv_batch b;
    const void * q;
    void * out;
    int64_t ldq, ldo;
    int32_t q_type, out_type, group, causal, window;
    float scale2;          // scale log2 e, scale > 0
    float cap2, cap_e;     // softcap log2 e (0: none), 2 log2 e scale / softcap
    float sign;            // q is multiplied by it: -1 for a negative scale, 0 for a scale of 0 (scale is then 1)
    int32_t chunk_cols;    // sequences of more columns than this are attend_chunk's
    float * partial;
    float * chunk_partial;
    int32_t chunk_blocks, chunk_splits;
};

// Tokens [lo, hi) that any of a sequence's rows i0 .. i1 sees.
__device__ inline void seen_by(const attn_args & a, const kv_seq & s, int i0, int i1, int32_t & lo, int32_t & hi) {
    const int32_t p0 = s.len - s.n + i0, p1 = s.len - s.n + i1;
    hi = a.causal ? min(s.len, max(0, p1 + 1)) : s.len;
    lo = a.window > 0 ? (int32_t) max((int64_t) 0, (int64_t) p0 - a.window + 1) : 0;
    lo = min(lo, hi);
}

// Units of work of one column tile of attend_few: whole UNITs from the first
// token that any of the sequence's rows sees.
__device__ inline int32_t units_of(const attn_args & a, const kv_seq & s) {
    int32_t lo, hi;
    seen_by(a, s, 0, s.n - 1, lo, hi);
    lo &= ~(GROUP - 1);
    return max(1, (hi - lo + UNIT - 1) / UNIT);
}

__device__ inline int32_t col_tiles(const attn_args & a, const kv_seq & s, int cols) { return (s.n * a.group + cols - 1) / cols; }

__device__ inline int32_t cost_of(const attn_args & a, const kv_seq & s, int cols) {
    return s.n > 0 && (int64_t) s.n * a.group <= a.chunk_cols ? units_of(a, s) * col_tiles(a, s, cols) * a.c.kv_heads : 0;
}

// A value of the lane's partner in the other half of the wave, and in the other
// 16 lanes of its half.
__device__ inline float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

__device__ inline float other_row(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 16) ? r[0] : r[1]);
}

// Query fragments of one column: 8 values each at d = at0, at0 + step, ..., from a
// row of any type, rounded to the cache's; zeros for a column past the last.
template <int TYPE, int N>
__device__ inline void load_q(const attn_args & a, const kv_seq & s, int D, int h, int c, bool valid, int at0, int step,
                              typename elem<TYPE>::frag qf[N]) {
    const int i = c / a.group, g = c - i * a.group;
    const int64_t at = (int64_t) (s.row0 + i) * a.ldq + (int64_t) (h * a.group + g) * D + at0;
#pragma unroll
    for (int k = 0; k < N; k++) {
        typename elem<TYPE>::frag f = {};
        if (valid) {
            if (a.q_type == TYPE) {
                f = *reinterpret_cast<const typename elem<TYPE>::frag *>((const uint16_t *) a.q + at + k * step);
            } else if (a.q_type == ZEST_TYPE_F32) {
                const float * x = (const float *) a.q + at + k * step;
                const float4 u = *reinterpret_cast<const float4 *>(x), w = *reinterpret_cast<const float4 *>(x + 4);
                const float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = elem<TYPE>::from(v[j]);
            } else if (a.q_type == ZEST_TYPE_BF16) {
                const bf16x8 x = *reinterpret_cast<const bf16x8 *>((const uint16_t *) a.q + at + k * step);
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = elem<TYPE>::from((float) x[j]);
            } else {
                const f16x8 x = *reinterpret_cast<const f16x8 *>((const uint16_t *) a.q + at + k * step);
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = elem<TYPE>::from((float) x[j]);
            }
            if (a.sign != 1.0f) {
#pragma unroll
                for (int j = 0; j < 8; j++) f[j] = elem<TYPE>::from((float) f[j] * a.sign);
            }
        }
        qf[k] = f;
    }
}

// Whether any of a fragment's values is NaN or infinite (an exponent field of
// ones carries into the next bit).
template <int TYPE> __device__ inline bool nonfinite(typename elem<TYPE>::frag f) {
    struct words { uint32_t w[4]; };
    const words v = __builtin_bit_cast(words, f);
    uint32_t carry = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) carry |= (v.w[i] & elem<TYPE>::EXP) + elem<TYPE>::ONE;
    return (carry & 0x80008000u) != 0;
}

// A weight of 0 does not silence a NaN or an infinity of V, so where a column may
// not see a token that holds one, V is split: `clean` has zeros for them and goes
// the usual way, `marks` has powers of 64 by their kind (1: +inf, 64: -inf, 4096:
// NaN; 0 for finite values), whose product with the columns' ones and zeros of
// the tokens they see counts each kind exactly (at most 32 of each).
template <int TYPE>
__device__ inline void split_nonfinite(typename elem<TYPE>::frag f, typename elem<TYPE>::frag & clean, typename elem<TYPE>::frag & marks) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    u16x8 v = __builtin_bit_cast(u16x8, f);
    constexpr unsigned short EXP = elem<TYPE>::EXP & 0xffffu;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const unsigned short w = v[i];
        const bool odd = (w & EXP) == EXP;
        marks[i] = elem<TYPE>::from(!odd ? 0.0f : (w & 0x7fff) != EXP ? 4096.0f : w >> 15 ? 64.0f : 1.0f);
        v[i] = odd ? 0 : w;
    }
    clean = __builtin_bit_cast(typename elem<TYPE>::frag, v);
}

// What such a count adds to a sum.
__device__ inline float counted(float n) {
    const int k = (int) n;
    const float pos = k & 63 ? INFINITY : 0.0f, neg = k >> 6 & 63 ? -INFINITY : 0.0f;
    return k >> 12 ? NAN : pos + neg;
}

// Four values of an output row.
__device__ inline void store4(const attn_args & a, int64_t at, const float v[4]) {
    if (a.out_type == ZEST_TYPE_F32) {
        *reinterpret_cast<float4 *>((float *) a.out + at) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
    uint16_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = a.out_type == ZEST_TYPE_BF16 ? __builtin_bit_cast(uint16_t, (__bf16) v[i]) : __builtin_bit_cast(uint16_t, (_Float16) v[i]);
    *reinterpret_cast<uint2 *>((uint16_t *) a.out + at) = make_uint2(w[0] | (uint32_t) w[1] << 16, w[2] | (uint32_t) w[3] << 16);
}

// Scores with a softcap, in units of log2: cap * tanh(x) as 1 - 2 / (e^2x + 1),
// off by 2^-22 of the cap at most.
__device__ inline float capped(const attn_args & a, float s) {
    return a.cap2 - 2.0f * a.cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s * a.cap_e) + 1.0f);
}

// That is 2^-16 of a score's unit at a cap of 64, less than a weight's rounding to
// 16 bits. From there on it would pass it, so scores below a quarter of the cap
// are multiplied by the series of tanh(x) / x (to x^8: off by 2^-26), which leaves
// an error of 2^-20 of the score at any cap. Not for all caps, as a chunk pays for
// it: 32 heads of 128, 2048 tokens at 8192, 311 us at a cap of 30, 380 at 100 (a
// decoding batch 165 and 166).
constexpr float PLAIN_CAP = 64.0f;

__device__ inline float capped_below(const attn_args & a, float s) {
    const float e = s * a.cap_e, y = e * e;          // e = 2 log2 e x
    constexpr float R = 0.25f / (LOG2E * LOG2E);     // x^2 / y
    const float q = fmaf(y, fmaf(y, fmaf(y, fmaf(y, R * R * R * R * 62.0f / 2835.0f, -R * R * R * 17.0f / 315.0f), R * R * 2.0f / 15.0f),
                                 -R / 3.0f), 1.0f);
    return fabsf(e) < 0.5f * LOG2E ? s * a.scale2 * q : capped(a, s);
}

template <typename V, int N> __device__ inline void cap_all(const attn_args & a, V & s) {
    if (a.cap2 > PLAIN_CAP * LOG2E) {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = capped_below(a, s[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = capped(a, s[i]);
    }
}

// A word that no wave changes while the kernel runs, at an address that is the
// same in every lane: a scalar load, which does not wait behind the direct loads
// in flight.
__device__ inline int32_t load_uniform(const int32_t * p) {
    return *(const __attribute__((address_space(4))) int32_t *) (uintptr_t) p;
}

// ---- few columns: decoding ----------------------------------------------------------

typedef __attribute__((address_space(3))) void * lds_ptr_t;
typedef const __attribute__((address_space(1))) void * global_ptr_t;

// The call's units are shared out evenly: the first total % W workgroups of W
// take one more than the others.
struct unit_shares {
    int32_t each, more;
    __device__ unit_shares(int32_t total, int W) : each(total / W), more(total - total / W * W) {}
    __device__ int32_t start(int w) const { return w * each + min(w, more); }
    __device__ int32_t owner(int32_t u) const {
        const int32_t big = more * (each + 1);
        return u < big ? u / (each + 1) : more + (u - big) / max(each, 1);
    }
};

// Tokens' K, then V, that a wave has in flight: RING_B steps of 32.
template <int D> constexpr int RING_B = D <= 64 ? 2 : 1;
template <int D> constexpr int STEP_BYTES = GROUP * D * 4;  // 32 tokens' K, then V
// A partial result of a column tile: O^T relative to the maxima, by columns, the
// maxima and the sums.
constexpr int partial_floats(int cols, int D) { return cols * (D + 2); }

// The units of every (sequence, k/v head, column tile) follow each other, and
// each workgroup takes an equal share of them, however long each sequence is. A
// piece of a share is one column tile's run of units; its four waves take 32
// tokens of a unit each and are joined in shared memory. A piece that is the
// tile's whole run goes to the output; else it is a partial result (slot 2w + 1
// where it starts the run, 2w where it continues one), and combine_few joins a
// run's pieces in order.
//
// HBM bound: 4 D bytes of K and V a token for 4 D COLS operations. A wave keeps a
// ring of its own in shared memory that direct loads fill (16 bytes a lane, whole
// kilobytes, no registers): K of the step to come is requested as soon as the
// scores are made, V as soon as it is weighed, and only this wave waits for them,
// by counting its loads. Eight waves a CU so have 64 to 128 KB in flight: 64
// sequences of 256 to 8192 tokens, 32 query and 8 k/v heads of 128, 104 us, 535 MB
// at 5.1 TB/s, where a large copy reaches 5.2 (with K and V loaded to registers
// 149 us); 4 of 20000 to 40000 with 5 new tokens and 48 heads 102 us.
//
// Tiles of 16 columns on v_mfma_f32_16x16x32, NT of them sharing the K and V read:
// a token's group of query heads rarely fills 32 columns, and half the columns
// are half the registers. The two 16-token score tiles of a step are tokens
// {0..7, 16..23} and {8..15, 24..31}, so that a lane group's 8 weights, in the
// registers they are in, are the 8 tokens of a V piece.
template <int TYPE, int D, int NT>
__device__ __forceinline__ void attend_few(const attn_args & a, int block, int blocks, uint8_t * ring_sh) {
    typedef typename elem<TYPE>::frag frag;
    constexpr int COLS = 16 * NT, KS = D / 32, DT = D / 16, R = RING_B<D>, LOADS = D / 16;  // loads of K (or V) a step
    // ring_sh, a wave: [R][K: D/8][32][8], V: [4][D][8]; then the prefix sums
    __shared__ float stat[WAVES][2][COLS];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lg = lane >> 4, col = lane & 15;
    const int ps = a.c.page_shift, P = 1 << ps;
    const zest::seq_index index(a.b, ps, reinterpret_cast<int32_t *>(ring_sh + WAVES * R * STEP_BYTES<D>),
                                [&](const kv_seq & s) { return cost_of(a, s, COLS); });
    const unit_shares shares(index.total, blocks);
    int32_t u = shares.start(block);
    const int32_t u1 = shares.start(block + 1);
    uint8_t * const mine = ring_sh + wave * R * STEP_BYTES<D>;
    const uint32_t ring_at = (uint32_t) (uintptr_t) (lds_ptr_t) mine;
    bool bad = false;
    while (u < u1) {
        int32_t before;
        const kv_seq s = index.at(u, before);
        const int32_t run = units_of(a, s), at = u - before, tiles = col_tiles(a, s, COLS);
        const int32_t item = at / run, first = at - item * run, h = item / tiles, ct = item - h * tiles;
        const int32_t units = min(run - first, u1 - u);
        const int32_t * row = a.b.tables + (int64_t) s.slot * a.b.table_cols;
        const int ncols = s.n * a.group, c0 = ct * COLS;
        // what all the tile's columns see, and what any of them does
        int32_t all_lo, all_hi, any_lo, any_hi, seq_lo, seq_hi;
        seen_by(a, s, c0 / a.group, c0 / a.group, any_lo, all_hi);
        const int last_row = (min(ncols, c0 + COLS) - 1) / a.group;
        seen_by(a, s, last_row, last_row, all_lo, any_hi);
        seen_by(a, s, 0, s.n - 1, seq_lo, seq_hi);
        const int32_t from = seq_lo;  // 16 tokens before it need no page: a window may have left them
        seq_lo &= ~(GROUP - 1);

        // this wave's steps: tokens t_first + j * UNIT .. + 31, j < n
        const int32_t t_first = seq_lo + first * UNIT + wave * GROUP;
        const int32_t n = min(units, max(0, (any_hi - t_first + UNIT - 1) / UNIT));
        const int64_t head_at = (int64_t) h * (4 * P * D);
        // the pages of a step's two 16-token halves (0 where there is none), and
        // which halves have one: bit g
        auto pages_of = [&](int j, int32_t id[2]) {
            uint32_t there = 0;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const int32_t t = t_first + j * UNIT + 16 * g;
                id[g] = 0;
                if (j < n && t < any_hi && t + 16 > from) {
                    const int32_t x = load_uniform(row + (t >> ps));
                    if ((uint32_t) x < (uint32_t) a.c.pages) {
                        id[g] = x;
                        there |= 1u << g;
                    } else {
                        bad = true;
                    }
                }
            }
            return there;
        };
        auto load_k = [&](int j, const int32_t id[2]) {
            const int32_t t0 = t_first + j * UNIT;
            const uint32_t in0 = t0 & (P - 1), in1 = (t0 + 16) & (P - 1);
            // a lane's token lane % 32 of K's rows 2i + lane / 32
            const int64_t off0 = id[0] * a.c.page_bytes + in0 * 16, off1 = id[1] * a.c.page_bytes + in1 * 16;
            const uint8_t * from = a.c.pool + head_at + (lane & 16 ? off1 : off0) + (lane & 15) * 16 + (lane >> 5) * (P * 16);
            const uint32_t to = ring_at + (j % R) * STEP_BYTES<D>;
#pragma unroll
            for (int i = 0; i < LOADS; i++)
                __builtin_amdgcn_global_load_lds((global_ptr_t) (from + i * (P * 32)), (lds_ptr_t) (uintptr_t) (to + i * 1024), 16, 0, 0);
        };
        auto load_v = [&](int j, const int32_t id[2]) {
            const int32_t t0 = t_first + j * UNIT;
            const uint32_t to = ring_at + (j % R) * STEP_BYTES<D> + GROUP * D * 2;
#pragma unroll
            for (int g = 0; g < 2; g++) {
                const uint32_t in = (t0 + 16 * g) & (P - 1);
                const uint8_t * from = a.c.pool + head_at + id[g] * a.c.page_bytes + 2 * P * D + in * (2 * D) + lane * 16;
#pragma unroll
                for (int i = 0; i < LOADS / 2; i++)
                    __builtin_amdgcn_global_load_lds((global_ptr_t) (from + i * 1024),
                                                     (lds_ptr_t) (uintptr_t) (to + (g * (LOADS / 2) + i) * 1024), 16, 0, 0);
            }
        };
        int32_t id[R + 1][2];      // of steps j .. j + R
        uint32_t there[R + 1];
#pragma unroll
        for (int r = 0; r < R; r++) {
            there[r] = pages_of(r, id[r]);
            if (r < n) {  // in this order: the waits below count on it
                load_k(r, id[r]);
                asm volatile("" ::: "memory");
                load_v(r, id[r]);
                asm volatile("" ::: "memory");
            }
        }

        frag qf[NT][KS];
        int32_t see_lo[NT], see_hi[NT];
#pragma unroll
        for (int q = 0; q < NT; q++) {
            const int c = c0 + 16 * q + col;
            load_q<TYPE, KS>(a, s, D, h, c, c < ncols, lg * 8, 32, qf[q]);
            seen_by(a, s, c / a.group, c / a.group, see_lo[q], see_hi[q]);
            if (c >= ncols) see_lo[q] = see_hi[q] = 0;
        }
        float m[NT], l[NT];
        f32x4 o[DT][NT];
#pragma unroll
        for (int q = 0; q < NT; q++) {
            m[q] = -INFINITY;
            l[q] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) o[dt][q] = f32x4{};
        }
        for (int32_t j = 0; j < n; j++) {
            const int32_t t0 = t_first + j * UNIT;
            uint8_t * const slot = mine + (j % R) * STEP_BYTES<D>;
            const bool more = j + R < n;
            there[R] = pages_of(j + R, id[R]);
            const bool masked = t0 < all_lo || t0 + GROUP > all_hi || there[0] != 3;

            // K: all but the loads after it
            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((2 * R - 1) * LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            f32x4 sc[NT][2];
#pragma unroll
            for (int q = 0; q < NT; q++) sc[q][0] = sc[q][1] = f32x4{};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int tok = (col & 7) + 16 * (col >> 3) + 8 * x;
                    const frag k = *reinterpret_cast<const frag *>(slot + ((ks * 4 + lg) * 32 + tok) * 16);
#pragma unroll
                    for (int q = 0; q < NT; q++) sc[q][x] = elem<TYPE>::mfma16(k, qf[q][ks], sc[q][x]);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K is read before it is overwritten
            if (more) load_k(j + R, id[R]);

            const float c = a.cap2 > 0.0f ? 1.0f : a.scale2;
            frag pf[NT];
#pragma unroll
            for (int q = 0; q < NT; q++) {
                // value e of x: token t0 + base + e + 8x of the lane group's base
                const int32_t base_t = t0 + 4 * (lg & 1) + 16 * (lg >> 1);
                if (a.cap2 > 0.0f) {
#pragma unroll
                    for (int x = 0; x < 2; x++) cap_all<f32x4, 4>(a, sc[q][x]);
                }
                if (masked) {
                    const bool page = there[0] >> (lg >> 1) & 1;
#pragma unroll
                    for (int x = 0; x < 2; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int32_t t = base_t + e + 8 * x;
                            sc[q][x][e] = page && t >= see_lo[q] && t < see_hi[q] ? sc[q][x][e] : -INFINITY;
                        }
                }
                float top = -INFINITY;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 4; e++) top = fmaxf(top, sc[q][x][e]);
                top = fmaxf(top, other_row(top));
                top = fmaxf(top, other_half(top)) * c;
                const float now = fmaxf(m[q], top);
                const float base = now == -INFINITY ? 0.0f : now;
                const float shrink = __builtin_amdgcn_exp2f(m[q] - base), shift = elem<TYPE>::SHIFT - base;
                if (__any(now != m[q])) {
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) o[dt][q] *= shrink;
                }
                m[q] = now;
                // The weights are the matrix instruction's operand, so they are rounded to
                // its 16 bits, each off by half a step at most and independently of the
                // others; their sum is of the unrounded ones, in 32 bits. Against 64 bits
                // that makes a bf16 chunk's outputs off by 0.0021 to 0.0023 of their size
                // where their own rounding costs 0.0017, a decoding batch's by 0.0018 to
                // 0.0020. A second operand for what the rounding leaves would halve the rate
                // at which a chunk meets V.
                float sum = 0.0f;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float w = __builtin_amdgcn_exp2f(fmaf(sc[q][x][e], c, shift));
                        sum += w;
                        pf[q][4 * x + e] = elem<TYPE>::from(w);
                    }
                l[q] = l[q] * shrink + sum;
            }

            if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((2 * R - 1) * LOADS) : "memory");
            else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            uint8_t * vp = slot + GROUP * D * 2 + (lg * D + col) * 16;
            bool odd = false;
            if (masked) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++) odd |= nonfinite<TYPE>(*reinterpret_cast<const frag *>(vp + dt * 256));
            }
            if (masked && __any(odd)) {
                frag seen[NT];
#pragma unroll
                for (int q = 0; q < NT; q++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int32_t t = t0 + 4 * (lg & 1) + 16 * (lg >> 1) + (e & 3) + 8 * (e >> 2);
                        const bool in = (there[0] >> (lg >> 1) & 1) && t >= see_lo[q] && t < see_hi[q];
                        seen[q][e] = elem<TYPE>::from(in ? 1.0f : 0.0f);
                    }
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    frag clean, marks;
                    split_nonfinite<TYPE>(*reinterpret_cast<const frag *>(vp + dt * 256), clean, marks);
                    *reinterpret_cast<frag *>(vp + dt * 256) = clean;  // the ring is this wave's own
#pragma unroll
                    for (int q = 0; q < NT; q++) {
                        const f32x4 n = elem<TYPE>::mfma16(marks, seen[q], f32x4{});
#pragma unroll
                        for (int i = 0; i < 4; i++) o[dt][q][i] += counted(n[i]);
                    }
                    asm volatile("" ::: "memory");
                    __builtin_amdgcn_sched_barrier(0);  // one block's registers serve the next
                }
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const frag v = *reinterpret_cast<const frag *>(vp + dt * 256);
#pragma unroll
                for (int q = 0; q < NT; q++) o[dt][q] = elem<TYPE>::mfma16(v, pf[q], o[dt][q]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) load_v(j + R, id[R]);
#pragma unroll
            for (int r = 0; r < R; r++) {
                there[r] = there[r + 1];
                id[r][0] = id[r + 1][0];
                id[r][1] = id[r + 1][1];
            }
        }

        // the waves' results joined: every column's maximum and sum, then O^T,
        // which each wave leaves in its ring by columns (units of 4 values, turned
        // by the column so that a wave's writes spread over the banks)
        constexpr int UNITS = D / 4;
#pragma unroll
        for (int q = 0; q < NT; q++) {
            l[q] += other_row(l[q]);
            l[q] += other_half(l[q]);
            if (lg == 0) {
                stat[wave][0][16 * q + col] = m[q];
                stat[wave][1][16 * q + col] = l[q];
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                int unit = 4 * dt + lg + col;
                if (unit >= UNITS) unit -= UNITS;
                *reinterpret_cast<f32x4 *>(mine + ((16 * q + col) * UNITS + unit) * 16) = o[dt][q];
            }
        }
        __syncthreads();
        const bool whole = units == run;
        float * part = a.partial + (int64_t) (2 * block + (first == 0)) * partial_floats(COLS, D);
        for (int i = threadIdx.x; i < COLS * UNITS; i += WAVES * 64) {
            const int oc = i / UNITS, unit = i - oc * UNITS;
            int turned = unit + (oc & 15);
            if (turned >= UNITS) turned -= UNITS;
            float top = stat[0][0][oc];
#pragma unroll
            for (int w = 1; w < WAVES; w++) top = fmaxf(top, stat[w][0][oc]);
            const float base = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float f = __builtin_amdgcn_exp2f(stat[w][0][oc] - base);
                const f32x4 x = *reinterpret_cast<const f32x4 *>(ring_sh + w * R * STEP_BYTES<D> + (oc * UNITS + turned) * 16);
                sum += stat[w][1][oc] * f;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] += x[e] * f;
            }
            const int cc = c0 + oc;
            if (!whole) {
                *reinterpret_cast<float4 *>(part + oc * D + unit * 4) = make_float4(v[0], v[1], v[2], v[3]);
                if (unit == 0) {
                    part[COLS * D + oc] = top;
                    part[COLS * D + COLS + oc] = sum;
                }
            } else if (cc < ncols) {
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] *= f;
                const int i0 = cc / a.group;
                store4(a, (int64_t) (s.row0 + i0) * a.ldo + (int64_t) (h * a.group + cc - i0 * a.group) * D + unit * 4, v);
            }
        }
        __syncthreads();
        u += units;
    }
    if (bad) zest::report(a.b.bad);
}

// Joins the pieces of the column tile whose run starts in workgroup w's share
// and goes on past it, if there is one: theirs are the last of the share. A
// workgroup takes 256 of the tile's groups of four values, the last one what is
// left (16 columns of 96 values are one and a half times 256), and requests eight
// pieces at a time.
template <int D, int NT> constexpr int COMBINE_PARTS = (16 * NT * D / 4 + 255) / 256;

template <int D, int NT> __device__ __forceinline__ void combine_few(const attn_args & a, int block, int part, int blocks, int32_t * attn_sh) {
    constexpr int COLS = 16 * NT, UNITS = D / 4;
    const zest::seq_index index(a.b, a.c.page_shift, attn_sh, [&](const kv_seq & s) { return cost_of(a, s, COLS); });
    const unit_shares shares(index.total, blocks);
    const int32_t u0 = shares.start(block), u1 = shares.start(block + 1);
    if (u0 == u1) return;
    int32_t before;
    const kv_seq s = index.at(u1 - 1, before);
    const int32_t run = units_of(a, s), at = u1 - 1 - before, tiles = col_tiles(a, s, COLS);
    // (costs that reached the sums' limit end there, with the last run cut short)
    const int32_t item = at / run, start = before + item * run, end = start + min(run, index.total - start);
    if (start < u0 || end <= u1) return;
    const int32_t h = item / tiles, ct = item - h * tiles, ncols = s.n * a.group;
    const int last = shares.owner(end - 1);
    {
        const int i = part * 256 + threadIdx.x, oc = i / UNITS, unit = i - oc * UNITS, cc = ct * COLS + oc;
        if (i >= COLS * UNITS || cc >= ncols) return;
        const float * x = a.partial + (int64_t) (2 * block + 1) * partial_floats(COLS, D);
        float m = x[COLS * D + oc], l = x[COLS * D + COLS + oc];
        float4 o = *reinterpret_cast<const float4 *>(x + oc * D + unit * 4);
        for (int w0 = block + 1; w0 <= last; w0 += 8) {
            float m1[8], l1[8];
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {  // past the last piece, that piece again, left out below
                const float * y = a.partial + (int64_t) (2 * min(w0 + k, last)) * partial_floats(COLS, D);
                m1[k] = y[COLS * D + oc];
                l1[k] = y[COLS * D + COLS + oc];
                v[k] = *reinterpret_cast<const float4 *>(y + oc * D + unit * 4);
            }
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const bool in = w0 + k <= last;
                const float now = in ? fmaxf(m, m1[k]) : m, base = now == -INFINITY ? 0.0f : now;
                const float f = __builtin_amdgcn_exp2f(m - base), g = __builtin_amdgcn_exp2f(m1[k] - base);
                m = now;
                const float4 x = make_float4(o.x * f + v[k].x * g, o.y * f + v[k].y * g, o.z * f + v[k].z * g, o.w * f + v[k].w * g);
                l = in ? l * f + l1[k] * g : l;
                o = make_float4(in ? x.x : o.x, in ? x.y : o.y, in ? x.z : o.z, in ? x.w : o.w);
            }
        }
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        const float v[4] = {o.x * f, o.y * f, o.z * f, o.w * f};
        const int i0 = cc / a.group;
        store4(a, (int64_t) (s.row0 + i0) * a.ldo + (int64_t) (h * a.group + cc - i0 * a.group) * D + unit * 4, v);
    }
}

// ---- chunks: many columns ---------------------------------------------------------

// Column tiles of 32 a wave of attend_chunk takes. Two would need 300 registers of
// a 128-wide head's wave, which leaves one wave a SIMD.
constexpr int QT = 1;
// Waves of a workgroup: eight where the rings leave room for one workgroup a CU
// and the registers for two waves a SIMD.
constexpr int chunk_waves(int D) { return D == 192 ? 8 : 4; }
template <int D> constexpr int CHUNK = chunk_waves(D) * 32 * QT;  // columns of a workgroup
// Steps of K and of V in shared memory. At step j the scores read K of j + 1 while
// those of j + 2 and j + 3 are on their way, the weights read V of j - 1.
constexpr int K_RING = 3, V_RING = 5;
template <int D> constexpr int CHUNK_RING = (K_RING + V_RING) * (STEP_BYTES<D> / 2);
// How far, in powers of two, a score may pass the maximum its column's weights
// are relative to before O^T is rescaled: the sums are in fp32, so only the
// weights' own range matters (bf16: fp32's; fp16: SHIFT + 8 stays below 2^16)
constexpr float SLACK = 8.0f;

template <int D> constexpr int CHUNK_PARTIAL = CHUNK<D> * (D + 2);

__device__ inline int32_t chunk_tiles_of(const attn_args & a, const kv_seq & s, int chunk) {
    const int64_t cols = (int64_t) s.n * a.group;
    return cols > a.chunk_cols ? (int32_t) ((cols + chunk - 1) / chunk) : 0;
}

// One column tile of a chunk: 4 or 8 waves of 32 QT columns each over the keys that
// any of the tile's columns sees, 32 tokens a step. K and V of a step go from
// the pool straight into shared memory (16 bytes a lane, in the pool's order,
// which is the order they are read in: every read is 512 contiguous bytes a half
// wave), two steps ahead of their use, with one barrier a step. A step runs three stages
// at once, so the matrix cores and the vector units both have work: the scores
// of step j + 1, the softmax of step j and the weights of step j - 1 times V.
//
// 32 query and 8 k/v heads of 128, the last 2048 of 8192 tokens: 255 to 266 us by
// card, 945 to 904 TFLOP/s, where a large library product reaches 1216. A step of a
// wave is 16 matrix instructions (512 cycles) and about 150 others; the board's
// power limit costs 12%, and leaving out the softmax or the loads would save 15%
// and 12%. On the way: K and V straight to registers, nothing shared, 891 us; one
// step ahead 289; two steps ahead 282, and without waiting for a page's number in
// every step and with a third of the address arithmetic 274; scores first in a
// step 261. Four waves of 32 columns, two workgroups a CU: 64 columns a wave halve
// the reads of shared memory (a third busy as it is) but leave one wave a SIMD.
// 192-wide heads take eight waves, one workgroup a CU: with four, a wave a SIMD,
// 765 us for 24 heads at 8192, with eight 342.
template <int TYPE, int D> __device__ __forceinline__ void attend_chunk(const attn_args & a, int block, int split, uint8_t * ring) {
    typedef typename elem<TYPE>::frag frag;
    constexpr int NQ = QT, KS = D / 16, DT = D / 32;
    // ring: [K_RING][D/8][32][8], [V_RING][2][2][D][8]; then the prefix sums
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5, col = lane & 31;
    const int ps = a.c.page_shift, P = 1 << ps;
    const zest::seq_index index(a.b, ps, reinterpret_cast<int32_t *>(ring + CHUNK_RING<D>),
                                [&](const kv_seq & s) { return chunk_tiles_of(a, s, CHUNK<D>); });
    // Under a causal mask the last tiles see the most. Where all fit the GPU at
    // once, two a CU, a CU gets one from either end (workgroup i + CUS joins i);
    // else the longest come first.
    const int h = block % a.c.kv_heads, order = block / a.c.kv_heads;
    // no more than the launch and the workspace are for: starts that go back make
    // sequences overlap (reported), and the tiles more than the rows allow
    const int total = min(index.total, a.chunk_blocks / a.c.kv_heads);
    int tile = total - 1 - order;
    if (tile < 0) return;
    if (total * a.c.kv_heads <= 2 * CUS) {
        const int head_start = CUS / a.c.kv_heads;
        if (order >= head_start) tile = order - head_start;
    }
    bool bad = false;
    int32_t before;
    const kv_seq s = index.at(tile, before);
    const int c0 = (tile - before) * CHUNK<D>, ncols = s.n * a.group;
    const int32_t * row = a.b.tables + (int64_t) s.slot * a.b.table_cols;

    // the tile's tokens, and of them this split's
    int32_t lo, hi;
    seen_by(a, s, c0 / a.group, min(ncols - 1, c0 + CHUNK<D> - 1) / a.group, lo, hi);
    const int32_t from = lo;  // pages wholly before it are not wanted: a window may have left them
    lo &= ~(GROUP - 1);
    const int32_t steps = (hi - lo + GROUP - 1) / GROUP;
    const int32_t first = (int32_t) ((int64_t) steps * split / a.chunk_splits);
    const int32_t n = (int32_t) ((int64_t) steps * (split + 1) / a.chunk_splits) - first;
    const int32_t t_first = lo + first * GROUP, t_hi = hi;

    // this wave's columns
    const int w0 = c0 + wave * 32 * NQ;
    frag qf[NQ][KS];
    int32_t see_lo[NQ], see_hi[NQ], all_lo = 0, all_hi = 0x7fffffff;
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const int c = w0 + 32 * q + col;
        load_q<TYPE, KS>(a, s, D, h, c, c < ncols, half * 8, 16, qf[q]);
        seen_by(a, s, c / a.group, c / a.group, see_lo[q], see_hi[q]);
        if (c >= ncols) see_lo[q] = see_hi[q] = 0;
    }
    if (w0 < ncols) {
        int32_t unused;
        seen_by(a, s, w0 / a.group, w0 / a.group, unused, all_hi);
        const int last = min(ncols, w0 + 32 * NQ) - 1;
        seen_by(a, s, last / a.group, last / a.group, all_lo, unused);
    }

    // The pages of 64 table columns, one a lane, so that a step's page is a lane
    // exchange: a load of it in the loop would wait behind the steps in flight.
    // absent: the columns without a page (bits; theirs is page 0, read and unseen).
    uint32_t window = 0;
    uint64_t absent = 0;
    int32_t at_col = 0;
    auto look_up = [&](int col0) {
        at_col = col0;
        const bool wanted = ((int64_t) (col0 + lane) << ps) < t_hi && ((int64_t) (col0 + lane + 1) << ps) > from;
        window = wanted ? (uint32_t) row[col0 + lane] : 0xffffffffu;
        const bool there = window < (uint32_t) a.c.pages;
        absent = __ballot(!there);
        bad |= wanted && !there;
        window = there ? window : 0;
        asm volatile("" : "+v"(window));  // waited for here, not at every use
    };
    look_up(t_first >> ps);
    // A step's loads: half of the waves make K's, half V's. Returns which 16 tokens
    // (bits) have no page. Few instructions, as a wave makes them every step: a
    // page's address is uniform, a lane's place in it one of the offsets made here.
    constexpr int CW = chunk_waves(D), LOADS = D / (8 * CW);  // loads a wave makes a step
    const bool k_wave = wave < CW / 2;
    const int v_first = (wave - CW / 2) * LOADS, v_group = v_first / (D / 32);  // of V's 2 D / 32 loads, and their 16 tokens
    const uint32_t page_bytes = (uint32_t) a.c.page_bytes;
    const uint32_t ring_at = (uint32_t) (uintptr_t) (lds_ptr_t) ring, v_ring_at = ring_at + K_RING * (STEP_BYTES<D> / 2);
    const uint8_t * const part = a.c.pool + (int64_t) h * (4 * P * D) + (k_wave ? 0 : 2 * P * D);
    uint32_t offset[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++)
        offset[i] = k_wave ? col * 16 + (2 * (wave * LOADS + i) + half) * (P * 16) : lane * 16 + (v_first + i) * 1024;
    auto load_step = [&](int j, int k_slot, int v_slot) -> uint32_t {
        if (j >= n) return 0;
        const int32_t t0 = t_first + j * GROUP;
        if (((t0 + 16) >> ps) - at_col >= 64) look_up(t0 >> ps);
        const int c0 = (t0 >> ps) - at_col;
        const uint32_t to = (k_wave ? ring_at + k_slot * (STEP_BYTES<D> / 2) + wave * LOADS * 1024
                                    : v_ring_at + v_slot * (STEP_BYTES<D> / 2) + v_first * 1024);
        const uint8_t * from = part + (uint64_t) (uint32_t) __builtin_amdgcn_readlane(window, c0) * page_bytes;
        uint32_t gone = absent >> c0 & 1 ? 3 : 0;
        if (ps == 4) {  // two pages a step
            const uint8_t * second = part + (uint64_t) (uint32_t) __builtin_amdgcn_readlane(window, c0 + 1) * page_bytes;
            gone = (uint32_t) (absent >> c0) & 3;
            const uint8_t * mine = k_wave ? (lane & 16 ? second - 256 : from) : v_group ? second - 32 * D : from;
#pragma unroll
            for (int i = 0; i < LOADS; i++)
                __builtin_amdgcn_global_load_lds((global_ptr_t) (mine + offset[i]), (lds_ptr_t) (uintptr_t) (to + i * 1024), 16, 0, 0);
        } else {
            from += (t0 & (P - 1)) * (k_wave ? 16 : 2 * D);
#pragma unroll
            for (int i = 0; i < LOADS; i++)
                __builtin_amdgcn_global_load_lds((global_ptr_t) (from + offset[i]), (lds_ptr_t) (uintptr_t) (to + i * 1024), 16, 0, 0);
        }
        return gone;
    };
    auto k_frag = [&](int slot, int ks) {
        return *reinterpret_cast<const frag *>(ring + slot * (STEP_BYTES<D> / 2) + (2 * ks + half) * 512 + col * 16);
    };
    auto v_frag = [&](int slot, int dt, int g) {
        return *reinterpret_cast<const frag *>(ring + (K_RING + slot) * (STEP_BYTES<D> / 2) + (2 * g + half) * (16 * D) + dt * 512 + col * 16);
    };

    f32x16 o[DT][NQ], s_cur[NQ], s_next[NQ];
    frag p[NQ][2];
    float m[NQ], l[NQ];
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        m[q] = -INFINITY;
        l[q] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt][q] = f32x16{};
    }
    auto scores = [&](int slot, f32x16 to[NQ]) {
#pragma unroll
        for (int q = 0; q < NQ; q++) to[q] = f32x16{};
#pragma unroll
        for (int ks = 0; ks < KS; ks++) {
            const frag k = k_frag(slot, ks);
#pragma unroll
            for (int q = 0; q < NQ; q++) to[q] = elem<TYPE>::mfma(k, qf[q][ks], to[q]);
        }
    };
    auto weigh = [&](int slot) {
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                const frag v = v_frag(slot, dt, g);
#pragma unroll
                for (int q = 0; q < NQ; q++) o[dt][q] = elem<TYPE>::mfma(v, p[q][g], o[dt][q]);
            }
    };
    // The same where a column does not see every token.
    auto weigh_masked = [&](int j, int slot, uint32_t gone) {
        bool odd = false;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int dt = 0; dt < DT; dt++) odd |= nonfinite<TYPE>(v_frag(slot, dt, g));
        if (!__any(odd)) {
            weigh(slot);
            return;
        }
#pragma unroll
        for (int g = 0; g < 2; g++) {
            frag seen[NQ];
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int32_t t = t_first + j * GROUP + 16 * g + 4 * half + (e & 3) + 8 * (e >> 2);
                    const bool in = t >= see_lo[q] && t < see_hi[q] && !(gone >> g & 1);
                    seen[q][e] = elem<TYPE>::from(in ? 1.0f : 0.0f);
                }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                frag clean, marks;
                split_nonfinite<TYPE>(v_frag(slot, dt, g), clean, marks);
#pragma unroll
                for (int q = 0; q < NQ; q++) {
                    const f32x16 n = elem<TYPE>::mfma(marks, seen[q], f32x16{});
                    o[dt][q] = elem<TYPE>::mfma(clean, p[q][g], o[dt][q]);
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][q][i] += counted(n[i]);
                }
                asm volatile("" ::: "memory");
                __builtin_amdgcn_sched_barrier(0);  // one block's registers serve the next
            }
        }
    };
    const float c = a.cap2 > 0.0f ? 1.0f : a.scale2;
    float shrink[NQ];
    // Maximum, sum and weights of s_cur; the weights go to `to`.
    auto soften = [&](frag to[NQ][2]) {
        bool any_rise = false;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            // (the weights' rounding: see attend_few's)
            float top = s_cur[q][0];
#pragma unroll
            for (int i = 1; i < 16; i++) top = fmaxf(top, s_cur[q][i]);
            top = fmaxf(top, other_half(top)) * c;
            // every column by itself, so that no row's result depends on others'
            const bool rise = top > m[q] + SLACK;
            any_rise |= rise;
            const float now = rise ? top : m[q];
            const float base = now == -INFINITY ? 0.0f : now;
            shrink[q] = __builtin_amdgcn_exp2f(m[q] - base);
            m[q] = now;
            const float shift = elem<TYPE>::SHIFT - base;
            float sum = 0.0f;
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(s_cur[q][8 * g + i], c, shift));
                    sum += w;
                    to[q][g][i] = elem<TYPE>::from(w);
                }
            l[q] = l[q] * shrink[q] + sum;
        }
        return any_rise;
    };

    // the steps that all of the wave's columns see whole
    const int whole_from = (max(all_lo - t_first, 0) + GROUP - 1) / GROUP, whole_to = (min(all_hi, t_hi) - t_first) / GROUP;
    // `gone` of the steps loaded, two bits each, the latest lowest
    uint32_t gones = load_step(0, 0, 0);
    gones = gones << 2 | load_step(1, 1, 1);
    gones = gones << 2 | load_step(2, 2, 2);
    int k_at = 0, v_at = 0;  // step j's places in the rings
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    bool masked_before = false;
    uint32_t gone_before = 0, gone = 0;
    // The barrier of step j: this wave's loads of step j + 1 are there (those of
    // j + 2 may not be) and its reads of step j - 1's scores and weights done;
    // past it, every wave's. Whether step j is masked.
    auto enter = [&](int j) {
        if (j + 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        gone = gones >> 4 & 3;
        gones = gones << 2 | load_step(j + 3, k_at, v_at >= 2 ? v_at - 2 : v_at + 3);
        return j < whole_from || j >= whole_to || gone != 0;
    };
    auto cap_scores = [&]() {
#pragma unroll
        for (int q = 0; q < NQ; q++) cap_all<f32x16, 16>(a, s_cur[q]);
    };
    auto finish = [&](bool rise, const frag pn[NQ][2]) {
        if (__any(rise)) {
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[dt][q][i] *= shrink[q];
        }
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            s_cur[q] = s_next[q];
            p[q][0] = pn[q][0];
            p[q][1] = pn[q][1];
        }
        k_at = k_at == K_RING - 1 ? 0 : k_at + 1;
        v_at = v_at == V_RING - 1 ? 0 : v_at + 1;
    };
    if (w0 >= ncols) {  // none of the tile's columns: this wave only loads
        for (int32_t j = 0; j < n; j++) {
            enter(j);
            k_at = k_at == K_RING - 1 ? 0 : k_at + 1;
            v_at = v_at == V_RING - 1 ? 0 : v_at + 1;
        }
        if (bad) zest::report(a.b.bad);
        return;
    }
    if (n > 0) scores(0, s_cur);
    auto k_next = [&]() { return k_at == K_RING - 1 ? 0 : k_at + 1; };
    auto v_last = [&]() { return v_at == 0 ? V_RING - 1 : v_at - 1; };
    int32_t j = 0;
    bool masked = n > 0 ? enter(0) : false;
    while (j < n) {
        // a step that is masked, or follows one that is, or the first
        if (a.cap2 > 0.0f) cap_scores();
        if (masked) {
            const int32_t t0 = t_first + j * GROUP;
#pragma unroll
            for (int q = 0; q < NQ; q++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int32_t t = t0 + (i & 3) + 8 * (i >> 2) + 4 * half;
                    const bool in = t >= see_lo[q] && t < see_hi[q] && !(gone >> (i >> 3) & 1);
                    s_cur[q][i] = in ? s_cur[q][i] : -INFINITY;
                }
        }
        {
            frag pn[NQ][2];
            if (j > 0) {
                if (masked_before) weigh_masked(j - 1, v_last(), gone_before);
                else weigh(v_last());
            }
            scores(k_next(), s_next);
            const bool rise = soften(pn);
            finish(rise, pn);
        }
        masked_before = masked;
        gone_before = gone;
        if (++j < n) masked = enter(j);
        // the steps that every column sees whole
        while (j < n && !masked && !masked_before) {
            if (a.cap2 > 0.0f) cap_scores();
            frag pn[NQ][2];
            scores(k_next(), s_next);
            weigh(v_last());
            const bool rise = soften(pn);
            // the weights are made here, beside the matrix instructions, not where
            // the next step first needs them
#pragma unroll
            for (int q = 0; q < NQ; q++) asm volatile("" : "+v"(pn[q][0]), "+v"(pn[q][1]), "+v"(l[q]));
            finish(rise, pn);
            if (++j < n) masked = enter(j);
        }
    }
    if (n > 0) {
        if (masked_before) weigh_masked(n - 1, v_last(), gone_before);
        else weigh(v_last());
    }
    if (bad) zest::report(a.b.bad);

    if (a.chunk_splits > 1) {
        // this split's part: O^T in the registers' own order, maxima and sums
        float * slot = a.chunk_partial + ((int64_t) (tile * a.c.kv_heads + h) * a.chunk_splits + split) * CHUNK_PARTIAL<D>;
#pragma unroll
        for (int q = 0; q < NQ; q++) {
            const int cc = wave * 32 * NQ + 32 * q;
            const float sum = l[q] + other_half(l[q]);
            if (half == 0) {
                slot[CHUNK<D> * D + cc + col] = m[q];
                slot[CHUNK<D> * (D + 1) + cc + col] = sum;
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    *reinterpret_cast<float4 *>(slot + cc * D + ((dt * 4 + k) * 64 + lane) * 4) =
                        make_float4(o[dt][q][4 * k], o[dt][q][4 * k + 1], o[dt][q][4 * k + 2], o[dt][q][4 * k + 3]);
        }
        return;
    }
#pragma unroll
    for (int q = 0; q < NQ; q++) {
        const float sum = l[q] + other_half(l[q]);
        const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
        const int cc = w0 + 32 * q + col;
        if (cc >= ncols) continue;
        const int64_t to = (int64_t) (s.row0 + cc / a.group) * a.ldo + (int64_t) (h * a.group + cc % a.group) * D + 4 * half;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float v[4] = {o[dt][q][4 * k] * f, o[dt][q][4 * k + 1] * f, o[dt][q][4 * k + 2] * f, o[dt][q][4 * k + 3] * f};
                store4(a, to + dt * 32 + 8 * k, v);
            }
    }
}

// Joins the splits of attend_chunk's column tiles, in their order: a workgroup a
// tile of 32 columns, a thread four values of each of its 32-row blocks.
template <int D> __device__ __forceinline__ void combine_chunk(const attn_args & a, int block, int32_t * attn_sh) {
    const zest::seq_index index(a.b, a.c.page_shift, attn_sh, [&](const kv_seq & s) { return chunk_tiles_of(a, s, CHUNK<D>); });
    constexpr int PARTS = CHUNK<D> / 32;
    const int part = block % PARTS, at = block / PARTS, h = at % a.c.kv_heads, tile = at / a.c.kv_heads;
    if (tile >= index.total) return;
    int32_t before;
    const kv_seq s = index.at(tile, before);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, k = threadIdx.x >> 6;
    const int cc = (tile - before) * CHUNK<D> + part * 32 + col;
    if (cc >= s.n * a.group) return;
    const float * slots = a.chunk_partial + (int64_t) at * a.chunk_splits * CHUNK_PARTIAL<D>;
    float m = -INFINITY, l = 0.0f;
#pragma unroll 8
    for (int i = 0; i < a.chunk_splits; i++) m = fmaxf(m, slots[(int64_t) i * CHUNK_PARTIAL<D> + CHUNK<D> * D + part * 32 + col]);
    const float base = m == -INFINITY ? 0.0f : m;
    float o[D / 32][4] = {};
    for (int i0 = 0; i0 < a.chunk_splits; i0 += 2) {
        float4 v[2][D / 32];
        float f[2], l1[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {  // past the last split, that split again, left out below
            const float * x = slots + (int64_t) min(i0 + e, a.chunk_splits - 1) * CHUNK_PARTIAL<D>;
            f[e] = x[CHUNK<D> * D + part * 32 + col];
            l1[e] = x[CHUNK<D> * (D + 1) + part * 32 + col];
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++) v[e][dt] = *reinterpret_cast<const float4 *>(x + part * 32 * D + ((dt * 4 + k) * 64 + lane) * 4);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const bool in = i0 + e < a.chunk_splits;
            const float w = __builtin_amdgcn_exp2f(f[e] - base);
            l = in ? l + l1[e] * w : l;
#pragma unroll
            for (int dt = 0; dt < D / 32; dt++) {
                const float x[4] = {v[e][dt].x, v[e][dt].y, v[e][dt].z, v[e][dt].w};
#pragma unroll
                for (int c = 0; c < 4; c++) o[dt][c] = in ? o[dt][c] + x[c] * w : o[dt][c];
            }
        }
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t to = (int64_t) (s.row0 + cc / a.group) * a.ldo + (int64_t) (h * a.group + cc % a.group) * D + 8 * k + 4 * half;
#pragma unroll
    for (int dt = 0; dt < D / 32; dt++) {
        const float v[4] = {o[dt][0] * f, o[dt][1] * f, o[dt][2] * f, o[dt][3] * f};
        store4(a, to + dt * 32, v);
    }
}

// ---- the kernels ----------------------------------------------------------------------

// The workgroups of few columns, then the chunks' (a.chunk_blocks of them, each in
// a.chunk_splits parts). A batch that holds both runs them side by side, one of
// the first a CU, as long as they last: they wait for memory while the others
// multiply. NT 0: none of few columns.
template <int TYPE, int D, int NT, bool CHUNKS>
__global__ __launch_bounds__((CHUNKS ? chunk_waves(D) : WAVES) * 64, D > 192 || (D > 128 && !CHUNKS) ? 1 : 2) void attn_kernel(attn_args a) {
    static_assert(!CHUNKS || NT == 0 || chunk_waves(D) == WAVES, "workgroups of one size");
    extern __shared__ __align__(1024) uint8_t smem[];
    const int few = gridDim.x - (CHUNKS ? a.chunk_blocks * a.chunk_splits : 0);
    if constexpr (CHUNKS)
        if ((int) blockIdx.x >= few) {
            const int at = blockIdx.x - few, split = at / a.chunk_blocks;
            attend_chunk<TYPE, D>(a, at - split * a.chunk_blocks, split, smem);
            return;
        }
    if constexpr (NT > 0) attend_few<TYPE, D, NT>(a, blockIdx.x, few, smem);
}

template <int D, int NT, bool CHUNKS> __global__ __launch_bounds__(256) void combine_kernel(attn_args a) {
    extern __shared__ __align__(16) int32_t attn_sh[];
    const int chunks = CHUNKS ? a.chunk_blocks * (CHUNK<D> / 32) : 0;
    if constexpr (CHUNKS)
        if ((int) blockIdx.x < chunks) {
            combine_chunk<D>(a, blockIdx.x, attn_sh);
            return;
        }
    if constexpr (NT > 0) {
        constexpr int PARTS = COMBINE_PARTS<D, NT>;
        const int at = blockIdx.x - chunks;
        combine_few<D, NT>(a, at / PARTS, at % PARTS, (gridDim.x - chunks) / PARTS, attn_sh);
    }
}

// ---- the host's plan ----------------------------------------------------------------

// What a call launches, by its sizes and bounds alone.
struct attn_plan {
    int64_t units, run;         // of attend_few, at most: in all, and of a column tile
    int workgroups, cols;       // of attend_few, 0: none; columns of its tiles
    int chunk_cols;             // sequences of more columns go to attend_chunk
    int64_t chunk_tiles;        // of attend_chunk, a k/v head, at most; 0: none
    int chunk_splits;
    size_t partial_bytes, bytes;
};

attn_plan plan_of(const zest_kv_cache * c, const zest_kv_batch * b, int group) {
    attn_plan p{};
    const int chunk = chunk_waves(c->head_dim) * 32;
    const int64_t most = (int64_t) b->max_new * group;  // columns of a sequence
    const int few_cols = most_few_cols(4.0 * b->seqs * b->max_len * c->kv_heads * c->head_dim);
    const bool chunks = most > few_cols;
    // one sequence alone is a chunk whatever its length turns out to be
    p.chunk_cols = !chunks ? 0x7fffffff : b->seqs == 1 ? 0 : few_cols;
    if (chunks) {
        p.chunk_tiles = std::min<int64_t>((b->rows * group + chunk - 1) / chunk + b->seqs, (most + chunk - 1) / chunk * b->seqs);
        // A tile's keys in the number of splits that keeps the CUs evenly busy:
        // rounds of workgroups times a split's steps, and the join's launch and
        // traffic (a step takes about 1.2 us, in which 6 MB are written or read
        // again). One sequence of 2048 tokens at 8192, 24 heads of 256: 384 tiles
        // on 256 CUs, in one part each 674 us, in two 566.
        const int64_t tiles = std::min<int64_t>(p.chunk_tiles, ((b->rows + b->seqs - 1) / b->seqs * group + chunk - 1) / chunk * b->seqs);
        const int64_t items = tiles * c->kv_heads, steps = b->max_len / GROUP + 1, slots = (c->head_dim <= 128 ? 2 : 1) * CUS;
        const double part = 8.0 * chunk * c->head_dim / 6e6;
        double best = 0;
        for (int64_t n = 1; n <= 64 && (n == 1 || (n <= steps / 8 && p.chunk_tiles * c->kv_heads * n <= 4 * slots)); n++) {
            const double cost = (double) ((items * n + slots - 1) / slots) * steps / n + (n > 1 ? 6.0 + part * items * n : 0.0);
            if (n == 1 || cost < best) {
                best = cost;
                p.chunk_splits = (int) n;
            }
        }
    }
    if (p.chunk_cols > 0) {
        const int64_t cols = std::min<int64_t>(most, p.chunk_cols);
        p.cols = cols <= 16 ? 16 : 32;
        p.run = std::max<int64_t>(1, ((int64_t) b->max_len + GROUP + UNIT - 1) / UNIT);
        const int64_t tiles = std::min<int64_t>((b->rows * group + p.cols - 1) / p.cols + b->seqs, (cols + p.cols - 1) / p.cols * b->seqs);
        p.units = p.run * tiles * c->kv_heads;
        p.workgroups = (int) std::min<int64_t>(p.units, c->head_dim <= 128 && !chunks ? 2 * CUS : CUS);
    }
    p.partial_bytes = (size_t) 2 * p.workgroups * partial_floats(p.cols, c->head_dim) * sizeof(float);
    p.bytes = p.partial_bytes;
    if (p.chunk_splits > 1) p.bytes += (size_t) p.chunk_tiles * c->kv_heads * p.chunk_splits * chunk * (c->head_dim + 2) * sizeof(float);
    p.bytes = std::max<size_t>(p.bytes, 16);
    return p;
}

// Lets a kernel have its ring and the largest prefix sums in shared memory, once a
// device (threads that launch it for the first time at once set the same value).
template <auto KERNEL> int allow_lds(size_t ring) {
    static std::atomic<uint64_t> set{0};  // a bit a device, those past the 64th every time
    int device = 0;
    if (const hipError_t e = hipGetDevice(&device); e != hipSuccess)
        return zest::fail(ZEST_E_HIP, "zest_kv_attn: current device: %s", hipGetErrorString(e));
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (set.load(std::memory_order_acquire) & bit) return ZEST_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize,
                                             (int) (ring + zest::seq_index_bytes(zest::KV_MAX_SEQS)));
    if (e != hipSuccess) return zest::fail(ZEST_E_HIP, "zest_kv_attn: shared memory attribute: %s", hipGetErrorString(e));
    set.fetch_or(bit, std::memory_order_release);
    return ZEST_OK;
}

template <int TYPE, int D, int NT, bool CHUNKS> int launch(attn_args & a, const attn_plan & p, hipStream_t s) {
    constexpr size_t few = NT ? WAVES * RING_B<D> * STEP_BYTES<D> : 0, ring = CHUNKS && CHUNK_RING<D> > few ? CHUNK_RING<D> : few;
    const size_t prefix = zest::seq_index_bytes(a.b.seqs);
    if (const int st = allow_lds<&attn_kernel<TYPE, D, NT, CHUNKS>>(ring)) return st;
    a.chunk_blocks = (int32_t) (p.chunk_tiles * a.c.kv_heads);
    hipLaunchKernelGGL((attn_kernel<TYPE, D, NT, CHUNKS>), dim3((unsigned) (a.chunk_blocks * p.chunk_splits + (NT ? p.workgroups : 0))),
                       dim3((CHUNKS ? chunk_waves(D) : WAVES) * 64), ring + prefix, s, a);
    // a run of one unit is never split, nor a chunk of one part
    constexpr int few_parts = NT ? COMBINE_PARTS<D, NT> : 1;
    const bool join_few = NT && p.run > 1, join_chunks = CHUNKS && p.chunk_splits > 1;
    if (join_chunks) {
        const unsigned blocks = (unsigned) (a.chunk_blocks * (CHUNK<D> / 32));
        hipLaunchKernelGGL((combine_kernel<D, NT, CHUNKS>), dim3(blocks + (join_few ? p.workgroups * few_parts : 0)), dim3(256), prefix, s, a);
    } else if (join_few) {
        hipLaunchKernelGGL((combine_kernel<D, NT, false>), dim3(p.workgroups * few_parts), dim3(256), prefix, s, a);
    }
    return zest::check_launch("zest_kv_attn");
}

template <int TYPE, int D> int launch(attn_args & a, const attn_plan & p, hipStream_t s) {
    if (p.chunk_tiles && p.workgroups) {
        if constexpr (chunk_waves(D) == WAVES) return launch<TYPE, D, 2, true>(a, p, s);
        attn_plan few = p;
        few.chunk_tiles = 0;
        few.chunk_splits = 0;
        if (const int st = launch<TYPE, D, 0, true>(a, p, s)) return st;
        return launch<TYPE, D, 2, false>(a, few, s);
    }
    if (p.chunk_tiles) return launch<TYPE, D, 0, true>(a, p, s);
    return p.cols == 16 ? launch<TYPE, D, 1, false>(a, p, s) : launch<TYPE, D, 2, false>(a, p, s);
}

template <int TYPE> int launch(attn_args & a, int D, const attn_plan & p, hipStream_t s) {
    switch (D) {
        case 64: return launch<TYPE, 64>(a, p, s);
        case 96: return launch<TYPE, 96>(a, p, s);
        case 128: return launch<TYPE, 128>(a, p, s);
        case 192: return launch<TYPE, 192>(a, p, s);
        default: return launch<TYPE, 256>(a, p, s);
    }
}

} // namespace

extern "C" {

size_t zest_kv_attn_workspace(const zest_kv_cache * cache, const zest_kv_batch * batch, int32_t q_heads) {
    if (!cache || !batch || cache->kv_heads <= 0 || q_heads < cache->kv_heads || q_heads % cache->kv_heads) return 0;
    if (batch->rows <= 0 || batch->seqs <= 0 || batch->max_new <= 0 || batch->max_len < 0) return 0;
    return plan_of(cache, batch, q_heads / cache->kv_heads).bytes;
}

int zest_kv_attn(const zest_kv_cache * cache, const zest_kv_batch * batch, const void * q, int q_type, int64_t ldq,
                 int32_t q_heads, float scale, int causal, int32_t window, float softcap, void * out, int out_type, int64_t ldo,
                 void * workspace, size_t workspace_bytes, uint32_t * bad, void * stream) {
    const char * me = "zest_kv_attn";
    if (const int st = zest::kv_check_cache(cache, me)) return st;
    if (const int st = zest::kv_check_batch(cache, batch, me)) return st;
    ZEST_REQUIRE(q_heads > 0 && q_heads <= 4096 && q_heads % cache->kv_heads == 0, "%s: %d query heads for %d k/v heads", me,
                 q_heads, cache->kv_heads);
    const int64_t width = (int64_t) q_heads * cache->head_dim;
    if (const int st = zest::kv_check_rows(q_type, q, ldq, width, me, "q")) return st;
    if (const int st = zest::kv_check_rows(out_type, out, ldo, width, me, "out")) return st;
    ZEST_REQUIRE(scale - scale == 0.0f && window >= 0 && softcap >= 0.0f && softcap - softcap == 0.0f,
                 "%s: scale=%g window=%d softcap=%g", me, (double) scale, window, (double) softcap);
    // (its quotient with the scale, times 2 log2 e, is a 32-bit number too)
    ZEST_REQUIRE(softcap == 0.0f || (scale == 0.0f ? 1.0 : std::fabs(scale)) / (double) softcap < 1e38, "%s: softcap=%g for scale=%g", me, (double) softcap,
                 (double) scale);
    // (a tile's last column, past the rows' by less than a tile, is a 32-bit number too)
    ZEST_REQUIRE(batch->rows * (int64_t) (q_heads / cache->kv_heads) < (1ll << 31) - 512, "%s: %lld rows of %d heads", me,
                 (long long) batch->rows, q_heads);
    const size_t qs = zest::kv_type_bytes(q_type), os = zest::kv_type_bytes(out_type);
    ZEST_REQUIRE(zest::kv_rows_apart(q, ldq * qs, width * qs, out, ldo * os, width * os, batch->rows), "%s: out overlaps q", me);
    ZEST_REQUIRE(zest::kv_rows_apart(cache->pool, 0, cache->pages * zest_kv_page_bytes(cache), out, 0, ((batch->rows - 1) * ldo + width) * os, 1),
                 "%s: out overlaps the pool", me);
    const attn_plan plan = plan_of(cache, batch, q_heads / cache->kv_heads);
    ZEST_REQUIRE(plan.units < (1ll << 31) && plan.chunk_tiles * cache->kv_heads * std::max(1, plan.chunk_splits) < (1ll << 22), "%s: a batch of %lld units of work",
                 me, (long long) std::max(plan.units, plan.chunk_tiles));
    const size_t need = plan.bytes;
    ZEST_REQUIRE(workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 && workspace_bytes >= need,
                 "%s: workspace of %zu bytes, 16-byte aligned, wanted", me, need);
    attn_args a{};
    a.c = zest::kv_pages_of(cache);
    a.b = zest::kv_batch_of(batch, bad);
    a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo;
    a.q_type = q_type, a.out_type = out_type;
    a.group = q_heads / cache->kv_heads;
    a.causal = causal != 0, a.window = window;
    a.sign = scale > 0.0f ? 1.0f : scale < 0.0f ? -1.0f : 0.0f;
    const float by = scale == 0.0f ? 1.0f : std::fabs(scale);
    a.scale2 = by * LOG2E;
    if (softcap > 0.0f) {
        a.cap2 = softcap * LOG2E;
        a.cap_e = by / softcap * (2.0f * LOG2E);
    }
    a.chunk_cols = plan.chunk_cols;
    a.chunk_splits = plan.chunk_splits;
    a.partial = (float *) workspace;
    a.chunk_partial = (float *) ((uint8_t *) workspace + plan.partial_bytes);
    const hipStream_t s = zest::as_stream(stream);
    return cache->type == ZEST_TYPE_BF16 ? launch<ZEST_TYPE_BF16>(a, cache->head_dim, plan, s)
                                         : launch<ZEST_TYPE_F16>(a, cache->head_dim, plan, s);
}

} // extern "C"

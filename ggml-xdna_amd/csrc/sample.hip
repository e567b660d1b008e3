// The choice of the next token (include/zest/decode.h).
//
// Everything that a token depends on is exact or an integer: logits are ordered
// by a 32-bit key, and a weight exp((x - max) / T) is computed in 64 bits and
// rounded to a whole number of 2^-45, so that 2^18 of them sum without a rounding
// or an overflow in 64 bits, in any order. What top-k and top-p keep is a cut: all
// logits above a key and those equal to it up to an index. It is found by histograms,
// of counts or of weights, first by the distance from the largest logit, then, if need
// be, by digits of the key, until no more than a wave's lanes are left to compare.
//
// Rows of up to 8192 logits are one workgroup's, which holds them in registers.
// Longer ones are cut in parts of 4096, a workgroup each, and the call is HBM bound by
// one reading (the next ones come from the last-level cache): stats_kernel finds the
// parts' largest logits, weigh_kernel the parts' weights, or a histogram of them,
// border_kernel, a workgroup a row, draws or finds the bins among which the cut lies,
// and, where there is a top-k or a top-p, collect_kernel lists their logits and
// finish_kernel cuts and draws. (With the last workgroup of a row to finish going on by
// itself, in three launches, the fences that takes cost 300 us for 64 rows of 151936.) In us:
// one row of 151936 with a top-k and a top-p 3.9, 6.7, 6.4, 6.5 and 13.3, 64 rows with a top-p
// 11, 23, 8, 18 and 15 (the 64-bit series in the second), 256 of 16 bits with a min-p 26, 30 and 7
// (two readings at 2.6 to 3 TB/s).
#include <algorithm>

#include "zest/decode.h"
#include "zest_common.h"

namespace {

typedef unsigned long long u64;

constexpr int PART = 4096, THREADS = 256, MAX_PARTS = ZEST_SAMPLE_MAX_VOCAB / PART;
constexpr int BINS = 256, LIST = 8192;    // of a histogram; logits that finish_kernel holds
constexpr int ROW_THREADS = 1024;         // of the kernels that are a workgroup a row
static_assert(THREADS == BINS, "a thread a bin");
constexpr int BATCH = 256;                // rows that a workspace is for: more go in several launches
constexpr int SHORT = 2048, MIDDLE = 8192;  // longest rows of the two sizes of row_kernel

// What a row's workgroups leave each other.
struct row_state {
    u64 top[MAX_PARTS];      // the largest key, then ~index of its first place
    uint32_t low[MAX_PARTS]; // the smallest key above -infinity's (none: 2^32 - 1)
    u64 mass[MAX_PARTS];
    u64 goal;                // of weights, within the bins that are listed
    uint32_t listed;
    int32_t from, to, mode;  // the bins that are listed
    u64 list[LIST];          // keys and indices
};
enum { DONE, KEEP_K, KEEP_P, SLOW };

// A part's histogram.
struct part_bins {
    u64 mass[BINS];
    uint32_t count[BINS];
};

struct sample_args {
    const void * logits;
    int64_t ld;
    int32_t type, vocab, parts;
    const float * u, * temperature;
    const int32_t * top_k;
    const float * top_p, * min_p;
    int32_t * token;
    float * prob;
    row_state * rows;
    part_bins * bins;        // [row][part]
};

// Keys order as the values do; NaN below all, -0 as 0.
__device__ inline uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return x != x ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) { return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key); }
constexpr uint32_t KEY_MINUS_INF = 0x007fffffu;

__device__ inline float logit(const sample_args & a, int64_t row, int i) {
    const int64_t at = row * a.ld + i;
    if (a.type == ZEST_TYPE_F32) return ((const float *) a.logits)[at];
    if (a.type == ZEST_TYPE_BF16) return (float) ((const __bf16 *) a.logits)[at];
    return (float) ((const _Float16 *) a.logits)[at];
}

// Four logits from index i on, of which those from `end` on are NaN (never taken).
__device__ inline void logits4(const sample_args & a, int64_t row, int i, int end, float x[4]) {
    if (i + 4 <= end) {
        const int64_t at = row * a.ld + i;
        if (a.type == ZEST_TYPE_F32) {  // (rows need not be aligned to the load)
            float4 v;
            __builtin_memcpy(&v, (const float *) a.logits + at, 16);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            uint2 v;
            __builtin_memcpy(&v, (const uint16_t *) a.logits + at, 8);
            const uint32_t w[4] = {v.x & 0xffffu, v.x >> 16, v.y & 0xffffu, v.y >> 16};
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = a.type == ZEST_TYPE_BF16 ? __uint_as_float(w[e] << 16) : (float) __builtin_bit_cast(_Float16, (uint16_t) w[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] = i + e < end ? logit(a, row, i + e) : NAN;
}

// A row's parameters, as the definition reads them.
struct params {
    double scale, p, m, u;  // scale in powers of two; p 1, m 0: off
    float width, near;      // logits further than this below the largest have no weight, or less than min_p
    int k;                  // vocab: off
    bool greedy;
    template <typename W> __device__ bool fits(const W & w) const { return m == 0.0 || w.value() >= m; }  // min_p
};

__device__ inline params params_of(const sample_args & a, int64_t row) {
    params r;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.scale = 1.4426950408889634074 / (double) t;
    r.width = 32.0f * t;
    const float p = a.top_p ? a.top_p[row] : 1.0f, m = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    r.p = p < 1.0f ? fmax((double) p, 0.0) : 1.0;  // (a NaN is off)
    r.m = m > 0.0f ? fmin((double) m, 1.0) : 0.0;
    r.near = r.m > 0.0 ? fminf(1.0001f * t * (0.01f - __logf((float) r.m)), r.width) : r.width;
    r.u = u > 0.0f ? (double) u : 0.0;
    const int k = a.top_k ? a.top_k[row] : 0;
    r.k = k > 0 ? min(k, a.vocab) : a.vocab;
    return r;
}

// A logit's weight relative to the largest, s 2^n: 2^y by the series of e^(f ln 2) for
// the part of y within half a unit (to its 12th power: off by 2^-52 at most). Adding
// 1.5 2^52 leaves a sum's whole part in its low bits.
struct weight {
    double s;
    int n;
    __device__ double value() const { return s * __hiloint2double((1023 + n) << 20, 0); }
    // in whole numbers of 2^-45
    __device__ u64 whole() const {
        constexpr double TWO52 = 4503599627370496.0;
        return (u64) (__double_as_longlong(fma(s, __hiloint2double((1023 + 45 + n) << 20, 0), TWO52)) - __double_as_longlong(TWO52));
    }
};

__device__ inline weight weight_of(float x, float top, double scale) {
    if (x == top) return {1.0, 0};
    const double d = (double) x - (double) top;
    if (!(d * scale >= -60.0) || top == INFINITY) return {0.0, 0};  // (a NaN, an infinity: none)
    constexpr double MAGIC = 6755399441055744.0;
    const double t = fma(d, scale, MAGIC), f = fma(d, scale, MAGIC - t) * 0.69314718055994530942;
    double s = 1.0 / 479001600.0;
    s = fma(s, f, 1.0 / 39916800.0);
    s = fma(s, f, 1.0 / 3628800.0);
    s = fma(s, f, 1.0 / 362880.0);
    s = fma(s, f, 1.0 / 40320.0);
    s = fma(s, f, 1.0 / 5040.0);
    s = fma(s, f, 1.0 / 720.0);
    s = fma(s, f, 1.0 / 120.0);
    s = fma(s, f, 1.0 / 24.0);
    s = fma(s, f, 1.0 / 6.0);
    s = fma(s, f, 0.5);
    s = fma(s, f, 1.0);
    s = fma(s, f, 1.0);
    return {s, (int) (uint32_t) __double_as_longlong(t)};
}
__device__ inline u64 whole(const weight & w) { return w.whole(); }

// ---- sums over a workgroup -----------------------------------------------------------

template <int N> struct group_memory {
    u64 wave[N / 64];
    u64 mass[BINS];
    uint32_t count[BINS];
    u64 rest, one;           // of the goal, within the digit that is left
    uint32_t digit, left;    // and the logits in it
    uint32_t listed;
    uint32_t keys[64], indices[64];
    u64 weights[64];
    uint32_t key;
    int32_t index;
};

template <typename V> __device__ inline V wave_sum(V v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

// The sum, in every thread; and the largest.
template <int N> __device__ inline u64 group_sum(group_memory<N> & sh, u64 v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 sum = 0;
#pragma unroll
    for (int w = 0; w < N / 64; w++) sum += sh.wave[w];
    return sum;
}
template <int N> __device__ inline u64 group_max(group_memory<N> & sh, u64 v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v = max(v, (u64) __shfl_xor(v, off));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < N / 64; w++) v = max(v, sh.wave[w]);
    return v;
}

__device__ inline u64 wave_upto(u64 v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 left = __shfl_up(v, off);
        if (lane >= off) v += left;
    }
    return v;
}

// What the threads before this one hold, and the workgroup's sum.
template <int N> __device__ inline u64 group_before(group_memory<N> & sh, u64 v, u64 & sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const u64 incl = wave_upto(v);
    __syncthreads();
    if (lane == 63) sh.wave[wave] = incl;
    __syncthreads();
    u64 before = incl - v;
    sum = 0;
#pragma unroll
    for (int w = 0; w < N / 64; w++) {
        if (w < wave) before += sh.wave[w];
        sum += sh.wave[w];
    }
    return before;
}

// Logits with a key above `key`, and those with that key up to `index`.
struct cut {
    uint32_t key;
    int32_t index;
    __device__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= index); }
};
constexpr cut EVERYTHING = {0, 0x7fffffff};

// Bins of equal width below `origin`, the last for all that is further away.
struct scale_of {
    float origin, per;
    __device__ int operator()(float x) const {
        if (x >= origin) return 0;
        const float d = (origin - x) * per;
        return d < (float) (BINS - 1) ? (int) d : BINS - 1;  // (a NaN: the last)
    }
    // from the largest logit to the smallest, or as far as there are weights
    static __device__ scale_of row(float top, float low, float width) {
        const float range = top == INFINITY ? 0.0f : fminf(top - low, width);
        return {top, range > 0.0f ? fminf((float) BINS / range, 3e38f) : 0.0f};
    }
};

// The cut behind which a running sum, from the largest logit on, first reaches `goal`
// (above 0): of counts, or of weights. `each` calls its argument with the key, the index
// and the weight of every logit that may be kept, in any order; where more than 64
// logits are equal at the cut, nth(key, r) is the index of the r-th of them (by index).
template <bool MASS, int N, typename Each, typename Nth> __device__ cut find_cut(group_memory<N> & sh, u64 goal, scale_of bins, Each each, Nth nth) {
    int bin = -1;          // of the distance; then digits of the key, from `shift` on
    uint32_t prefix = 0;
    int shift = 32;
    auto in = [&](uint32_t k) { return bin < 0 || (bins(value_of(k)) == bin && (shift == 32 || k >> shift == prefix >> shift)); };
    for (;;) {
        __syncthreads();
        for (int i = threadIdx.x; i < BINS; i += N) {
            sh.mass[i] = 0;
            sh.count[i] = 0;
        }
        if (threadIdx.x == 0) sh.listed = 0;
        __syncthreads();
        each([&](uint32_t k, int, u64 w) {
            if (!in(k)) return;
            const int d = bin < 0 ? bins(value_of(k)) : 255 - (int) (k >> (shift - 8) & 255);  // the largest first
            if (MASS) atomicAdd(&sh.mass[d], w);
            atomicAdd(&sh.count[d], 1u);
        });
        __syncthreads();
        if (threadIdx.x < 64) {  // four bins a lane
            u64 here[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                here[i] = MASS ? sh.mass[4 * threadIdx.x + i] : sh.count[4 * threadIdx.x + i];
                sum += here[i];
            }
            const u64 upto = wave_upto(sum), all = __shfl(upto, 63);
            goal = min(goal, all);  // (a product of the total may be rounded past it)
            if (upto >= goal && upto - sum < goal) {
                u64 above = upto - sum;
                int d = 0;
#pragma unroll
                for (int i = 0; i < 3; i++) {
                    if (above + here[i] >= goal) break;
                    above += here[i];
                    d++;
                }
                sh.digit = 4 * threadIdx.x + d;
                sh.left = sh.count[4 * threadIdx.x + d];
                sh.rest = goal - above;
            }
        }
        __syncthreads();
        goal = sh.rest;
        if (bin < 0) {
            bin = (int) sh.digit;
        } else {
            shift -= 8;
            prefix |= (255 - sh.digit) << shift;
        }
        if (sh.left <= 64 || shift == 0) break;
    }
    if (sh.left <= 64) {
        each([&](uint32_t k, int i, u64 w) {
            if (!in(k)) return;
            const uint32_t at = atomicAdd(&sh.listed, 1u);
            sh.keys[at] = k;
            sh.indices[at] = (uint32_t) i;
            sh.weights[at] = MASS ? w : 1;
        });
        __syncthreads();
        const uint32_t n = sh.listed, lane = threadIdx.x;
        if (lane < n) {
            const uint32_t k = sh.keys[lane], i = sh.indices[lane];
            u64 before = 0;
            for (uint32_t j = 0; j < n; j++) before += sh.keys[j] > k || (sh.keys[j] == k && sh.indices[j] < i) ? sh.weights[j] : 0;
            if (before < goal && before + sh.weights[lane] >= goal) {
                sh.key = k;
                sh.index = (int) i;
            }
        }
        __syncthreads();
        const cut c{sh.key, sh.index};
        __syncthreads();
        return c;
    }
    // of the equal ones, as many as it takes
    if (MASS) {
        each([&](uint32_t k, int, u64 w) {
            if (k == prefix) sh.one = w;  // the same of all of them
        });
        __syncthreads();
        goal = (goal + sh.one - 1) / max(sh.one, (u64) 1);
    }
    return {prefix, nth(prefix, goal)};
}

// ---- short rows ----------------------------------------------------------------------

// A workgroup a row, E consecutive logits a thread: 8, since 16 of 1024 threads' take more
// registers than there are (120 spilled). Latency: 1003 logits with top-k, top-p
// and min-p take 12.8 us.
template <int N, int E> __global__ __launch_bounds__(N) void row_kernel(sample_args a) {
    __shared__ group_memory<N> sh;
    const int64_t row = blockIdx.x;
    const int first = threadIdx.x * E;
    float x[E];
#pragma unroll
    for (int i = 0; i < E; i += 4) logits4(a, row, first + i, a.vocab, x + i);
    const params p = params_of(a, row);
    u64 best = 0;
#pragma unroll
    for (int i = 0; i < E; i++) best = max(best, first + i < a.vocab ? (u64) key_of(x[i]) << 32 | (uint32_t) ~(first + i) : 0);
    best = group_max(sh, best);
    const uint32_t top_key = (uint32_t) (best >> 32);
    if (top_key <= KEY_MINUS_INF || p.greedy) {
        if (threadIdx.x == 0) {
            a.token[row] = top_key <= KEY_MINUS_INF ? -1 : (int32_t) ~(uint32_t) best;
            if (a.prob) a.prob[row] = top_key <= KEY_MINUS_INF ? 0.0f : 1.0f;
        }
        return;
    }
    const float top = value_of(top_key);
    u64 w[E];
    uint32_t fit = 0;  // those of at least min_p
#pragma unroll
    for (int i = 0; i < E; i++) {
        const weight v = weight_of(x[i], top, p.scale);
        w[i] = whole(v);
        fit |= (uint32_t) p.fits(v) << i;
    }
    u64 low = 0;  // the smallest key that has a weight, as the largest of the others' distances
#pragma unroll
    for (int i = 0; i < E; i++) low = max(low, w[i] ? (u64) (top_key - key_of(x[i])) : 0);
    const scale_of bins = scale_of::row(top, value_of(top_key - (uint32_t) group_max(sh, low)), p.width);
    cut c = EVERYTHING;
    auto each = [&](auto what) {
#pragma unroll
        for (int i = 0; i < E; i++) {
            const uint32_t k = key_of(x[i]);
            if (w[i] && c.keeps(k, first + i)) what(k, first + i, w[i]);
        }
    };
    auto nth = [&](uint32_t key, u64 r) {  // of one key, those that the cut so far keeps
        u64 n = 0, all;
        each([&](uint32_t k, int, u64) { n += k == key; });
        u64 before = group_before(sh, n, all);
        r = min(r, all);
        each([&](uint32_t k, int i, u64) {
            if (k == key && ++before == r) sh.index = i;
        });
        __syncthreads();
        return sh.index;
    };
    if (p.k < a.vocab) c = find_cut<false>(sh, (u64) p.k, bins, each, nth);
    if (p.p < 1.0) {
        u64 sum = 0;
        each([&](uint32_t, int, u64 v) { sum += v; });
        sum = group_sum(sh, sum);
        c = find_cut<true>(sh, max((u64) __builtin_ceil(p.p * (double) sum), (u64) 1), bins, each, nth);
    }
    u64 mine = 0, total;
    each([&](uint32_t, int i, u64 v) { mine += fit >> (i - first) & 1 ? v : 0; });
    u64 before = group_before(sh, mine, total);
    const u64 goal = min((u64) (p.u * (double) total), total - 1);
    if (before <= goal && goal < before + mine)
        each([&](uint32_t, int i, u64 v) {
            v = fit >> (i - first) & 1 ? v : 0;
            if (before <= goal && goal < before + v) {
                a.token[row] = i;
                if (a.prob) a.prob[row] = (float) ((double) v / (double) total);
            }
            before += v;
        });
}

// ---- long rows -----------------------------------------------------------------------

// A part of a row in a workgroup of N threads: logit e of step j is PART part + (j N +
// thread) 4 + e.
template <int N> __device__ inline int index_of(int part, int j) { return part * PART + (j * N + (int) threadIdx.x) * 4; }
template <int N> __device__ inline void load_part(const sample_args & a, int64_t row, int part, float x[PART / N / 4][4]) {
#pragma unroll
    for (int j = 0; j < PART / N / 4; j++) logits4(a, row, index_of<N>(part, j), a.vocab, x[j]);
}
constexpr int STEPS = PART / THREADS / 4;

struct row_top {
    float top;        // the largest logit
    scale_of bins;
    bool none;
    int32_t first;    // the largest one's first place
    __device__ row_top(const sample_args & a, const row_state & s, const params & p) {
        const int lane = threadIdx.x & 63;
        u64 t = lane < a.parts ? s.top[lane] : 0;
        uint32_t l = lane < a.parts ? s.low[lane] : 0xffffffffu;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            t = max(t, (u64) __shfl_xor(t, off));
            l = min(l, (uint32_t) __shfl_xor((int) l, off));
        }
        const uint32_t key = (uint32_t) (t >> 32);
        none = key <= KEY_MINUS_INF;
        top = value_of(key);
        first = (int32_t) ~(uint32_t) t;
        bins = none ? scale_of{0.0f, 0.0f} : scale_of::row(top, value_of(min(l, key)), p.width);
    }
};

__global__ __launch_bounds__(THREADS) void stats_kernel(sample_args a) {
    __shared__ group_memory<THREADS> sh;
    __shared__ uint32_t lows[THREADS / 64];
    const int part = blockIdx.x;
    const int64_t row = blockIdx.y;
    float x[STEPS][4];
    load_part<THREADS>(a, row, part, x);
    u64 best = 0;
    uint32_t low = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < STEPS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t k = key_of(x[j][e]);
            best = max(best, k ? (u64) k << 32 | (uint32_t) ~(index_of<THREADS>(part, j) + e) : 0);
            if (k > KEY_MINUS_INF) low = min(low, k);
        }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) low = min(low, (uint32_t) __shfl_xor((int) low, off));
    if ((threadIdx.x & 63) == 0) lows[threadIdx.x >> 6] = low;
    best = group_max(sh, best);
    row_state & s = a.rows[row];
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; w++) low = min(low, lows[w]);
        s.top[part] = best;
        s.low[part] = low;
        if (part == 0) s.listed = 0;
    }
}

// Whether a row has neither a top-k nor a top-p.
__device__ inline bool uncut(const sample_args & a, const params & p) { return p.k >= a.vocab && p.p >= 1.0; }

// Of each part the weights that min_p keeps or, where the row has a top-k or a top-p, a
// histogram of weights and counts by distance from the largest logit.
__global__ __launch_bounds__(THREADS) void weigh_kernel(sample_args a) {
    __shared__ group_memory<THREADS> sh;
    const int part = blockIdx.x;
    const int64_t row = blockIdx.y;
    row_state & s = a.rows[row];
    float x[STEPS][4];
    load_part<THREADS>(a, row, part, x);
    const params p = params_of(a, row);
    const row_top t(a, s, p);
    if (t.none || p.greedy) return;
    if (uncut(a, p)) {
        u64 sum = 0;
#pragma unroll
        for (int j = 0; j < STEPS; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (t.top - x[j][e] > p.near) continue;  // (most: a wave passes over the series)
                const weight w = weight_of(x[j][e], t.top, p.scale);
                sum += p.fits(w) ? whole(w) : 0;
            }
        sum = group_sum(sh, sum);
        if (threadIdx.x == 0) s.mass[part] = sum;
        return;
    }
    for (int i = threadIdx.x; i < BINS; i += THREADS) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < STEPS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const u64 w = whole(weight_of(x[j][e], t.top, p.scale));
            if (w) {
                const int b = t.bins(x[j][e]);
                atomicAdd(&sh.mass[b], w);
                atomicAdd(&sh.count[b], 1u);
            }
        }
    __syncthreads();
    part_bins & bins = a.bins[row * a.parts + part];
    for (int i = threadIdx.x; i < BINS; i += THREADS) {
        bins.mass[i] = sh.mass[i];
        bins.count[i] = sh.count[i];
    }
}

// The draw: the part in which u lies by the parts' weights, then the logit, of those that
// the cut and min_p keep.
template <int N> __device__ void draw(group_memory<N> & sh, const sample_args & a, int64_t row, const params & p, float top, cut c, const u64 * mass) {
    const int lane = threadIdx.x & 63;
    const u64 upto = wave_upto(lane < a.parts ? mass[lane] : 0), total = __shfl(upto, 63);
    const u64 goal = min((u64) (p.u * (double) total), total - 1);
    const int part = __popcll(__ballot(upto <= goal));
    u64 run = part ? __shfl(upto, max(part - 1, 0)) : 0;
    float x[PART / N / 4][4];
    load_part<N>(a, row, part, x);
#pragma unroll
    for (int j = 0; j < PART / N / 4; j++) {
        u64 w[4], mine = 0, sum;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const weight v = weight_of(x[j][e], top, p.scale);
            w[e] = p.fits(v) && c.keeps(key_of(x[j][e]), index_of<N>(part, j) + e) ? whole(v) : 0;
            mine += w[e];
        }
        u64 before = run + group_before(sh, mine, sum);
        run += sum;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if (before <= goal && goal < before + w[e]) {
                a.token[row] = index_of<N>(part, j) + e;
                if (a.prob) a.prob[row] = (float) ((double) w[e] / (double) total);
            }
            before += w[e];
        }
    }
}

// Rows without a cut drawn; of the others the bins among which it lies.
__global__ __launch_bounds__(ROW_THREADS) void border_kernel(sample_args a) {
    __shared__ group_memory<ROW_THREADS> sh;
    const int64_t row = blockIdx.x;
    row_state & s = a.rows[row];
    const params p = params_of(a, row);
    const row_top t(a, s, p);
    if (t.none || p.greedy) {
        if (threadIdx.x == 0) {
            a.token[row] = t.none ? -1 : t.first;
            if (a.prob) a.prob[row] = t.none ? 0.0f : 1.0f;
            s.mode = DONE;
        }
        return;
    }
    if (uncut(a, p)) {
        if (threadIdx.x == 0) s.mode = DONE;
        draw(sh, a, row, p, t.top, EVERYTHING, s.mass);
        return;
    }
    // the parts' bins, every fourth part a quarter of the threads
    const int i = threadIdx.x % BINS, q0 = threadIdx.x / BINS;
    if (q0 == 0) sh.mass[i] = sh.count[i] = 0;
    __syncthreads();
    u64 m = 0;
    uint32_t n = 0;
#pragma unroll 4
    for (int q = q0; q < a.parts; q += ROW_THREADS / BINS) {
        m += a.bins[row * a.parts + q].mass[i];
        n += a.bins[row * a.parts + q].count[i];
    }
    atomicAdd(&sh.mass[i], m);
    atomicAdd(&sh.count[i], n);
    __syncthreads();
    m = q0 == 0 ? sh.mass[i] : 0;
    n = q0 == 0 ? sh.count[i] : 0;
    u64 all_mass, all_count;
    const u64 mass_before = group_before(sh, m, all_mass), count_before = group_before(sh, (u64) n, all_count);
    const bool by_k = (u64) p.k < all_count;  // (top-k keeps all there is otherwise)
    if (!by_k && p.p >= 1.0) {
        if (threadIdx.x == 0) s.mode = KEEP_P, s.from = BINS, s.to = -1, s.goal = 0;  // everything, nothing listed
        return;
    }
    const u64 goal = by_k ? (u64) p.k : min(max((u64) __builtin_ceil(p.p * (double) all_mass), (u64) 1), all_mass);
    const u64 before = by_k ? count_before : mass_before, here = by_k ? (u64) n : m;
    if (before < goal && before + here >= goal) {
        s.mode = (by_k ? count_before + n : n) > LIST ? SLOW : by_k ? KEEP_K : KEEP_P;
        s.from = by_k ? 0 : i;
        s.to = i;
        s.goal = goal - (by_k ? 0 : before);
    }
}

// The logits of the bins among which the cut lies, into the row's list, and of the parts
// the weights above them.
__global__ __launch_bounds__(THREADS) void collect_kernel(sample_args a) {
    __shared__ group_memory<THREADS> sh;
    __shared__ uint32_t at;
    const int part = blockIdx.x;
    const int64_t row = blockIdx.y;
    row_state & s = a.rows[row];
    const int mode = s.mode, from = s.from, to = s.to;
    if (mode == DONE || mode == SLOW) return;
    float x[STEPS][4];
    load_part<THREADS>(a, row, part, x);
    const params p = params_of(a, row);
    const row_top t(a, s, p);
    if (threadIdx.x == 0) at = 0;
    __syncthreads();
    // before the last bin all have a weight: they are nearer than 255 / 256 width, where it is
    // e^-31.875 > 2^-46 at least (unless bins cannot be as narrow as the width asks)
    const bool fine = t.bins.per < 3e38f;
    u64 above = 0;
    uint32_t mine = 0, place[STEPS][4];
#pragma unroll
    for (int j = 0; j < STEPS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int b = t.bins(x[j][e]);
            place[j][e] = 0xffffffffu;
            if (b < from && p.m > 0.0 && !(t.top - x[j][e] > p.near)) {
                const weight w = weight_of(x[j][e], t.top, p.scale);
                above += p.fits(w) ? whole(w) : 0;
            } else if (b >= from && b <= to && ((fine && b < BINS - 1) || whole(weight_of(x[j][e], t.top, p.scale)))) {
                place[j][e] = atomicAdd(&at, 1u);
            }
        }
    if (p.m == 0.0 && (int) threadIdx.x < from) above = a.bins[row * a.parts + part].mass[threadIdx.x];
    __syncthreads();
    if (threadIdx.x == 0) mine = at ? atomicAdd(&s.listed, at) : 0;
    above = group_sum(sh, above);
    if (threadIdx.x == 0) {
        s.mass[part] = above;
        at = mine;
    }
    __syncthreads();
    mine = at;
#pragma unroll
    for (int j = 0; j < STEPS; j++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (place[j][e] != 0xffffffffu && mine + place[j][e] < LIST)
                s.list[mine + place[j][e]] = (u64) key_of(x[j][e]) << 32 | (uint32_t) (index_of<THREADS>(part, j) + e);
}

// The cut and the draw. A row whose cut lies among more logits than a list holds (very
// many equal ones, or a top-k of thousands) is read itself for every histogram.
__global__ __launch_bounds__(ROW_THREADS) void finish_kernel(sample_args a) {
    __shared__ group_memory<ROW_THREADS> sh;
    __shared__ u64 list[LIST], mass[MAX_PARTS];
    const int64_t row = blockIdx.x;
    row_state & s = a.rows[row];
    const int mode = s.mode;
    if (mode == DONE) return;
    const params p = params_of(a, row);
    const row_top t(a, s, p);
    cut c = EVERYTHING;
    const bool listed = mode != SLOW;
    const int n = listed ? min((int) s.listed, LIST) : a.vocab;
    if (listed)
        for (int i = threadIdx.x; i < n; i += ROW_THREADS) list[i] = s.list[i];
    for (int q = threadIdx.x; q < a.parts; q += ROW_THREADS) mass[q] = mode == KEEP_P ? s.mass[q] : 0;
    __syncthreads();
    if (n > 0) {
        auto each = [&](auto what) {
            for (int i = threadIdx.x; i < n; i += ROW_THREADS) {
                const uint32_t k = listed ? (uint32_t) (list[i] >> 32) : key_of(logit(a, row, i));
                const int index = listed ? (int) (uint32_t) list[i] : i;
                if (!c.keeps(k, index)) continue;
                const u64 w = whole(weight_of(value_of(k), t.top, p.scale));
                if (w) what(k, index, w);
            }
        };
        // (in no order: the r-th place of a key has r - 1 of its places before it)
        auto nth = [&](uint32_t key, u64 r) {
            u64 ties = 0;
            each([&](uint32_t k, int, u64) { ties += k == key; });
            ties = group_sum(sh, ties);
            if (r >= ties) return 0x7fffffff;
            int lo = -1, hi = a.vocab;  // at or before lo there are less than r, at or before hi r
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                u64 some = 0;
                each([&](uint32_t k, int i, u64) { some += k == key && i <= mid; });
                if (group_sum(sh, some) >= r) hi = mid;
                else lo = mid;
            }
            return hi;
        };
        // the histogram's bins are those of what is listed
        scale_of bins = t.bins;
        if (listed) {
            bins.origin -= bins.per > 0.0f ? (float) s.from / bins.per : 0.0f;
            bins.per = fminf(bins.per * ((float) BINS / (float) (s.to - s.from + 1)), 3e38f);
        }
        const bool by_k = mode == KEEP_K || (!listed && p.k < a.vocab);
        if (by_k) c = find_cut<false>(sh, (u64) p.k, bins, each, nth);
        if (p.p < 1.0) {
            u64 goal = s.goal;
            if (mode != KEEP_P) {
                u64 sum = 0;
                each([&](uint32_t, int, u64 w) { sum += w; });
                goal = max((u64) __builtin_ceil(p.p * (double) group_sum(sh, sum)), (u64) 1);
            }
            c = find_cut<true>(sh, goal, bins, each, nth);
        }
        each([&](uint32_t k, int i, u64 w) {
            if (p.fits(weight_of(value_of(k), t.top, p.scale))) atomicAdd(&mass[i / PART], w);
        });
        __syncthreads();
    }
    draw(sh, a, row, p, t.top, c, mass);
}

size_t bins_bytes(int64_t rows, int64_t parts) { return (size_t) rows * parts * sizeof(part_bins); }

} // namespace

extern "C" {

size_t zest_sample_workspace(int64_t rows, int64_t vocab) {
    if (rows <= 0 || rows > 65536 || vocab <= 0 || vocab > ZEST_SAMPLE_MAX_VOCAB || vocab <= MIDDLE) return 0;
    rows = std::min<int64_t>(rows, BATCH);
    return (size_t) rows * sizeof(row_state) + bins_bytes(rows, (vocab + PART - 1) / PART);
}

int zest_sample(const void * logits, int type, int64_t rows, int64_t vocab, int64_t ld, const float * u, const float * temperature,
                const int32_t * top_k, const float * top_p, const float * min_p, int32_t * token, float * prob, void * workspace,
                size_t workspace_bytes, void * stream) {
    const char * me = "zest_sample";
    if (type != ZEST_TYPE_F32 && type != ZEST_TYPE_F16 && type != ZEST_TYPE_BF16)
        return zest::fail(ZEST_E_UNSUPPORTED, "%s: logits of type %d (F32, F16 or BF16)", me, type);
    ZEST_REQUIRE(rows > 0 && rows <= 65536 && vocab > 0 && vocab <= ZEST_SAMPLE_MAX_VOCAB, "%s: %lld rows of %lld logits", me, (long long) rows,
                 (long long) vocab);
    ZEST_REQUIRE(logits && u && token, "%s: null pointer", me);
    const uintptr_t size = type == ZEST_TYPE_F32 ? 4 : 2;
    ZEST_REQUIRE(reinterpret_cast<uintptr_t>(logits) % size == 0 && (rows == 1 || (ld >= vocab && ld < (1ll << 31))), "%s: misaligned logits or ld=%lld", me,
                 (long long) ld);
    for (const void * p : {(const void *) u, (const void *) temperature, (const void *) top_k, (const void *) top_p, (const void *) min_p,
                           (const void *) token, (const void *) prob})
        ZEST_REQUIRE(reinterpret_cast<uintptr_t>(p) % 4 == 0, "%s: parameters and results 4-byte aligned wanted", me);
    const size_t need = zest_sample_workspace(rows, vocab);
    ZEST_REQUIRE(!need || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= need),
                 "%s: workspace of %zu bytes, 16-byte aligned, wanted", me, need);
    sample_args a{};
    a.logits = logits;
    a.ld = rows == 1 ? vocab : ld;
    a.type = type;
    a.vocab = (int32_t) vocab;
    a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.token = token, a.prob = prob;
    const hipStream_t s = zest::as_stream(stream);
    if (vocab <= SHORT) {
        hipLaunchKernelGGL((row_kernel<256, SHORT / 256>), dim3((unsigned) rows), dim3(256), 0, s, a);
        return zest::check_launch(me);
    }
    if (vocab <= MIDDLE) {
        hipLaunchKernelGGL((row_kernel<1024, MIDDLE / 1024>), dim3((unsigned) rows), dim3(1024), 0, s, a);
        return zest::check_launch(me);
    }
    a.parts = (int32_t) ((vocab + PART - 1) / PART);
    a.rows = (row_state *) workspace;
    a.bins = (part_bins *) ((uint8_t *) workspace + std::min<int64_t>(rows, BATCH) * sizeof(row_state));
    for (int64_t r0 = 0; r0 < rows; r0 += BATCH) {
        const dim3 grid((unsigned) a.parts, (unsigned) std::min<int64_t>(rows - r0, BATCH));
        hipLaunchKernelGGL(stats_kernel, grid, dim3(THREADS), 0, s, a);
        hipLaunchKernelGGL(weigh_kernel, grid, dim3(THREADS), 0, s, a);
        hipLaunchKernelGGL(border_kernel, dim3(grid.y), dim3(ROW_THREADS), 0, s, a);
        if (top_k || top_p) {
            hipLaunchKernelGGL(collect_kernel, grid, dim3(THREADS), 0, s, a);
            hipLaunchKernelGGL(finish_kernel, dim3(grid.y), dim3(ROW_THREADS), 0, s, a);
        }
        if (const int st = zest::check_launch(me)) return st;
        a.logits = (const uint8_t *) a.logits + BATCH * a.ld * size;
        a.u += BATCH, a.token += BATCH;
        for (const float ** q : {&a.temperature, &a.top_p, &a.min_p}) *q = *q ? *q + BATCH : nullptr;
        a.top_k = a.top_k ? a.top_k + BATCH : nullptr;
        a.prob = a.prob ? a.prob + BATCH : nullptr;
    }
    return ZEST_OK;
}

} // extern "C"

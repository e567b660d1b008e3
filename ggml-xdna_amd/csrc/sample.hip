// The choice of the next token (include/zest/decode.h).
//
// Everything that a token depends on is exact or an integer: logits are ordered
// by a 32-bit key, and a weight exp((x - max) / T) is computed in 64 bits and
// rounded to a whole number of 2^-45, so that 2^18 of them sum without a rounding
// or an overflow in 64 bits, in any order. What top-k and top-p keep is a cut: all
// logits above a key and the first few, by index, of those equal to it.
#include <algorithm>

#include "zest/decode.h"
#include "zest_common.h"

namespace {

typedef __bf16 bf16_t;
typedef unsigned long long u64;

constexpr double ONE = 35184372088832.0;  // 2^45: the largest weight
constexpr int THREADS = 1024, WAVES = THREADS / 64;

struct sample_args {
    const void * logits;
    int64_t ld;
    int32_t type, vocab;
    const float * u, * temperature;
    const int32_t * top_k;
    const float * top_p, * min_p;
    int32_t * token;
    float * prob;
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
    if (a.type == ZEST_TYPE_BF16) return (float) ((const bf16_t *) a.logits)[at];
    return (float) ((const _Float16 *) a.logits)[at];
}

// A row's parameters, as the definition reads them.
struct params {
    double scale, p, m, u;  // p 1, m 0: off
    int k;                  // vocab: off
    bool greedy;
};

__device__ inline params params_of(const sample_args & a, int64_t row) {
    params r;
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    r.greedy = !(t > 0.0f);
    r.scale = 1.0 / (double) t;
    const float p = a.top_p ? a.top_p[row] : 1.0f, m = a.min_p ? a.min_p[row] : 0.0f, u = a.u[row];
    r.p = p < 1.0f ? fmax((double) p, 0.0) : 1.0;  // (a NaN is off)
    r.m = m > 0.0f ? fmin((double) m, 1.0) : 0.0;
    r.u = u > 0.0f ? (double) u : 0.0;
    const int k = a.top_k ? a.top_k[row] : 0;
    r.k = k > 0 ? min(k, a.vocab) : a.vocab;
    return r;
}

// A logit's weight relative to the largest, and as an integer.
__device__ inline double weight_of(float x, float top, double scale) {
    if (x == top) return 1.0;
    return x > -INFINITY && top < INFINITY ? exp(((double) x - (double) top) * scale) : 0.0;  // (a NaN: 0)
}
__device__ inline u64 whole(double w) { return (u64) __builtin_rint(w * ONE); }

// ---- one workgroup a row -----------------------------------------------------------

__device__ inline u64 wave_sum(u64 v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

struct shared_row {
    u64 wave[WAVES];
    u64 mass[256];
    uint32_t count[256];
    u64 found;
    uint32_t key;
};

// The sum over the workgroup, in every thread.
__device__ inline u64 group_sum(shared_row & sh, u64 v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 sum = 0;
    for (int w = 0; w < WAVES; w++) sum += sh.wave[w];
    return sum;
}

// What the threads before this one hold, and the workgroup's sum.
__device__ inline u64 group_before(shared_row & sh, u64 v, u64 & sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 incl = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 left = __shfl_up(incl, off);
        if (lane >= off) incl += left;
    }
    __syncthreads();
    if (lane == 63) sh.wave[wave] = incl;
    __syncthreads();
    u64 before = incl - v;
    sum = 0;
    for (int w = 0; w < WAVES; w++) {
        if (w < wave) before += sh.wave[w];
        sum += sh.wave[w];
    }
    return before;
}

// Logits with a key above `key`, and the first `ties` with that key.
struct cut {
    uint32_t key, ties;
};

// The cut behind which a running sum, from the largest logit on, reaches `goal`:
// of counts (MASS false) or weights, over the logits above `in`. Eight bits of the
// key at a time, from the top: a histogram of the logits that agree so far.
template <bool MASS>
__device__ cut find_cut(shared_row & sh, const sample_args & a, int64_t row, float top, double scale, cut in, double goal) {
    uint32_t prefix = 0;
    u64 above = 0;  // sum over the keys above the prefix's
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += THREADS) {
            sh.mass[i] = 0;
            sh.count[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
            const float x = logit(a, row, i);
            const uint32_t k = key_of(x);
            if (k < in.key || (shift < 24 && (k >> (shift + 8)) != prefix >> (shift + 8))) continue;
            atomicAdd(&sh.count[k >> shift & 255], 1u);
            if (MASS && k != in.key) atomicAdd(&sh.mass[k >> shift & 255], whole(weight_of(x, top, scale)));
        }
        __syncthreads();
        // ties at `in` count as far as it keeps them
        if (MASS && threadIdx.x == 0 && (shift == 24 || (in.key >> (shift + 8)) == prefix >> (shift + 8)) && in.key > KEY_MINUS_INF)
            sh.mass[in.key >> shift & 255] += in.ties * whole(weight_of(value_of(in.key), top, scale));
        __syncthreads();
        if (threadIdx.x == 0) {
            int d = 255;
            for (; d > 0; d--) {
                const u64 here = MASS ? sh.mass[d] : sh.count[d];
                if ((double) (above + here) >= goal) break;
                above += here;
            }
            // (where no sum reaches it the last digit with anything stays)
            sh.found = above;
            sh.key = prefix | (uint32_t) d << shift;
        }
        __syncthreads();
        above = sh.found;
        prefix = sh.key;
    }
    cut r{prefix, 0};
    uint32_t have = sh.count[prefix & 255];
    if (prefix == in.key) have = min(have, in.ties);
    if (MASS) {
        const u64 one = prefix > KEY_MINUS_INF ? whole(weight_of(value_of(prefix), top, scale)) : 0;
        // the first of them is kept if what lies above does not reach the goal
        const double left = goal - (double) above;
        r.ties = one == 0 ? have : (uint32_t) fmin(fmax(ceil(left / (double) one), 1.0), (double) have);
    } else {
        r.ties = (uint32_t) min((u64) have, (u64) goal - above);
    }
    return r;
}

__global__ __launch_bounds__(THREADS) void sample_kernel(sample_args a) {
    __shared__ shared_row sh;
    const int64_t row = blockIdx.x;
    const params p = params_of(a, row);
    // the largest logit and its first place
    u64 best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
        const u64 v = (u64) key_of(logit(a, row, i)) << 32 | (uint32_t) ~i;
        best = max(best, v);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) best = max(best, (u64) __shfl_xor(best, off));
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = best;
    __syncthreads();
    for (int w = 0; w < WAVES; w++) best = max(best, sh.wave[w]);
    const uint32_t top_key = (uint32_t) (best >> 32);
    if (top_key <= KEY_MINUS_INF || p.greedy) {
        if (threadIdx.x == 0) {
            a.token[row] = top_key <= KEY_MINUS_INF ? -1 : (int32_t) ~(uint32_t) best;
            if (a.prob) a.prob[row] = top_key <= KEY_MINUS_INF ? 0.0f : 1.0f;
        }
        return;
    }
    const float top = value_of(top_key);
    cut c{0, 0};
    if (p.k < a.vocab) c = find_cut<false>(sh, a, row, top, p.scale, c, (double) p.k);
    auto kept = [&](float x, uint32_t k, u64 tie) { return k > c.key || (k == c.key && tie < c.ties); };
    if (p.p < 1.0) {
        u64 sum = 0;
        for (int i = threadIdx.x; i < a.vocab; i += THREADS) {
            const float x = logit(a, row, i);
            if (key_of(x) > c.key) sum += whole(weight_of(x, top, p.scale));
        }
        sum = group_sum(sh, sum);
        if (c.key > KEY_MINUS_INF) sum += c.ties * whole(weight_of(value_of(c.key), top, p.scale));
        c = find_cut<true>(sh, a, row, top, p.scale, c, fmax(p.p * (double) sum, 1.0));
    }
    // What stays, in index order: first its sum, then the place that u points at.
    // (Which of the cut's ties stay goes by their rank, so they are counted along.)
    u64 total = 0, goal = 0;
    for (int pass = 0; pass < 2; pass++) {
        u64 run = 0, ties = 0;
        for (int i0 = 0; i0 < a.vocab; i0 += THREADS) {
            const int i = i0 + threadIdx.x;
            const float x = i < a.vocab ? logit(a, row, i) : -INFINITY;
            const uint32_t k = i < a.vocab ? key_of(x) : 0;
            u64 tie_sum;
            const u64 tie = ties + group_before(sh, k == c.key && i < a.vocab, tie_sum);
            ties += tie_sum;
            const double w = weight_of(x, top, p.scale);
            const u64 mine = i < a.vocab && kept(x, k, tie) && w >= p.m ? whole(w) : 0;
            u64 sum;
            const u64 before = run + group_before(sh, mine, sum);
            run += sum;
            if (pass == 1 && mine && before <= goal && goal < before + mine) {
                a.token[row] = i;
                if (a.prob) a.prob[row] = (float) ((double) mine / (double) total);
            }
        }
        total = run;
        goal = min((u64) (p.u * (double) total), total - 1);
    }
}

} // namespace

extern "C" {

size_t zest_sample_workspace(int64_t rows, int64_t vocab) {
    if (rows <= 0 || rows > 65536 || vocab <= 0 || vocab > ZEST_SAMPLE_MAX_VOCAB) return 0;
    return 16;
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
    ZEST_REQUIRE(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= need,
                 "%s: workspace of %zu bytes, 16-byte aligned, wanted", me, need);
    sample_args a{};
    a.logits = logits;
    a.ld = rows == 1 ? vocab : ld;
    a.type = type;
    a.vocab = (int32_t) vocab;
    a.u = u, a.temperature = temperature, a.top_k = top_k, a.top_p = top_p, a.min_p = min_p;
    a.token = token, a.prob = prob;
    hipLaunchKernelGGL(sample_kernel, dim3((unsigned) rows), dim3(THREADS), 0, zest::as_stream(stream), a);
    return zest::check_launch(me);
}

} // extern "C"

// Products of a few rows with GGUF weights as they are (include/zest/decode.h):
// y[m][n] = sum_k x[m][k] W[n][k], HBM bound by the weights' bytes.
//
// A chunk is 32 of a weight row's values, of which 16 bytes of codes hold two
// halves of 16: the low and the high nibbles (Q8_0: 32 bytes, its first and last
// 16). Every half is code * scale + offset, codes signed bytes.
#include <algorithm>
#include <atomic>

#include "kv_device.h"
#include "zest/decode.h"
#include "zest_common.h"
#include "zest_device.h"

namespace {

constexpr int MAX_M = ZEST_MATVEC_MAX_ROWS, MAX_N = ZEST_MATVEC_MAX_GROUP;

__device__ inline float half_to_float(uint32_t h) { return (float) __builtin_bit_cast(_Float16, (uint16_t) h); }

// Bytes of a row that need not be aligned to the load (the hardware takes any).
template <typename T> __device__ inline T load_as(const uint8_t * p) {
    T v;
    __builtin_memcpy(&v, p, sizeof(T));
    return v;
}

// The published levels of IQ4_NL and IQ4_XS, four codes (0..15, one a byte) at a
// time: two byte permutes look up the low and the high eight, bit 3 picks.
__device__ inline uint32_t iq4_levels(uint32_t n) {
    constexpr auto b = [](int v) { return (uint32_t) (v & 255); };
    constexpr auto four = [](int x, int y, int z, int w) { return (uint32_t) (x & 255) | (uint32_t) (y & 255) << 8 | (uint32_t) (z & 255) << 16 | (uint32_t) (w & 255) << 24; };
    constexpr uint32_t T0 = four(-127, -104, -83, -65), T1 = four(-49, -35, -22, -10), T2 = four(1, 13, 25, 38), T3 = four(53, 69, 89, 113);
    const uint32_t sel = n & 0x07070707u;
    const uint32_t lo = __builtin_amdgcn_perm(T1, T0, sel), hi = __builtin_amdgcn_perm(T3, T2, sel);
    const uint32_t m = ((n >> 3) & 0x01010101u) * 0xffu;
    return (hi & m) | (lo & ~m);
}

// Of a type: bytes of a block, chunks of a block, the loads of a chunk, and what
// they stand for.
template <int TYPE> struct quant;

// A chunk's halves: codes (four to a word) and w = scale * code + offset.
struct half_scales {
    float scale[2], offset[2];
};

// The first of a half's 16 columns, and the row's alignment.
template <int TYPE> __device__ inline int64_t half_column(int64_t chunk, int half) {
    if constexpr (TYPE == ZEST_TYPE_Q4_K) return chunk / 2 * 64 + chunk % 2 * 16 + half * 32;
    return chunk * 32 + half * 16;
}

constexpr int row_align(int type) {
    return type == ZEST_TYPE_Q4_K ? 16 : type == ZEST_TYPE_IQ4_XS ? 8 : type == ZEST_TYPE_Q4_1 ? 4 : 2;
}

// d, qs[16]: w = d (q - 8), or d level[q]
template <int TYPE> struct quant_nibbles {
    struct raw { uint4 q; uint32_t d; };
    static constexpr int BYTES = 18, CHUNKS = 1;
    static __device__ raw load(const uint8_t * row, int64_t chunk) {
        const uint8_t * p = row + chunk * BYTES;
        return {load_as<uint4>(p + 2), load_as<uint16_t>(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][4]) {
        const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (TYPE == ZEST_TYPE_Q4_0) {
                const uint32_t s = w[i] ^ 0x88888888u;  // 16 (q - 8), the nibble as a byte's high half
                c[0][i] = s << 4 & 0xf0f0f0f0u;
                c[1][i] = s & 0xf0f0f0f0u;
            } else {
                c[0][i] = iq4_levels(w[i] & 0x0f0f0f0fu);
                c[1][i] = iq4_levels(w[i] >> 4 & 0x0f0f0f0fu);
            }
        }
    }
    static __device__ half_scales scales(const raw & r, int64_t) {
        const float d = half_to_float(r.d) * (TYPE == ZEST_TYPE_Q4_0 ? 0.0625f : 1.0f);
        return {{d, d}, {0.0f, 0.0f}};
    }
};
template <> struct quant<ZEST_TYPE_Q4_0> : quant_nibbles<ZEST_TYPE_Q4_0> {};
template <> struct quant<ZEST_TYPE_IQ4_NL> : quant_nibbles<ZEST_TYPE_IQ4_NL> {};

// d, m, qs[16]: w = d q + m
template <> struct quant<ZEST_TYPE_Q4_1> {
    struct raw { uint4 q; uint32_t dm; };
    static constexpr int BYTES = 20, CHUNKS = 1;
    static __device__ raw load(const uint8_t * row, int64_t chunk) {
        const uint8_t * p = row + chunk * BYTES;
        return {load_as<uint4>(p + 4), load_as<uint32_t>(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][4]) {
        const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[0][i] = w[i] & 0x0f0f0f0fu;
            c[1][i] = w[i] >> 4 & 0x0f0f0f0fu;
        }
    }
    static __device__ half_scales scales(const raw & r, int64_t) {
        const float d = half_to_float(r.dm), m = half_to_float(r.dm >> 16);
        return {{d, d}, {m, m}};
    }
};

// d, qs[32]: w = d q
template <> struct quant<ZEST_TYPE_Q8_0> {
    struct raw { uint4 q[2]; uint32_t d; };
    static constexpr int BYTES = 34, CHUNKS = 1;
    static __device__ raw load(const uint8_t * row, int64_t chunk) {
        const uint8_t * p = row + chunk * BYTES;
        return {{load_as<uint4>(p + 2), load_as<uint4>(p + 18)}, load_as<uint16_t>(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][4]) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            c[h][0] = r.q[h].x;
            c[h][1] = r.q[h].y;
            c[h][2] = r.q[h].z;
            c[h][3] = r.q[h].w;
        }
    }
    static __device__ half_scales scales(const raw & r, int64_t) {
        const float d = half_to_float(r.d);
        return {{d, d}, {0.0f, 0.0f}};
    }
};

// d, dmin, 12 bytes of 6-bit scales and minima of 8 sub-blocks of 32, qs[128]: 64
// values to 32 bytes, sub-block 2r in the low nibbles, 2r + 1 in the high ones;
// w = d sc q - dmin m
template <> struct quant<ZEST_TYPE_Q4_K> {
    struct raw { uint4 q, head; };
    static constexpr int BYTES = 144, CHUNKS = 8;
    static __device__ raw load(const uint8_t * row, int64_t chunk) {
        const uint8_t * p = row + (chunk >> 3) * BYTES;
        return {*reinterpret_cast<const uint4 *>(p + 16 + (chunk & 7) * 16), *reinterpret_cast<const uint4 *>(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][4]) {
        const uint32_t w[4] = {r.q.x, r.q.y, r.q.z, r.q.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[0][i] = w[i] & 0x0f0f0f0fu;
            c[1][i] = w[i] >> 4 & 0x0f0f0f0fu;
        }
    }
    static __device__ half_scales scales(const raw & r, int64_t chunk) {
        const int run = (int) (chunk & 7) >> 1;  // sub-blocks 2 run and 2 run + 1
        const float d = half_to_float(r.head.x), dmin = half_to_float(r.head.x >> 16);
        // the first four sub-blocks' fields are low 6 bits, the others' 4 bits and the first's top two
        const bool far = run >= 2;
        const uint32_t sc = far ? (r.head.w & 0x0f0f0f0fu) | (r.head.y >> 2 & 0x30303030u) : r.head.y & 0x3f3f3f3fu;
        const uint32_t m = far ? (r.head.w >> 4 & 0x0f0f0f0fu) | (r.head.z >> 2 & 0x30303030u) : r.head.z & 0x3f3f3f3fu;
        const uint32_t s = sc >> 16 * (run & 1), n = m >> 16 * (run & 1);
        return {{d * (float) (s & 0xff), d * (float) (s >> 8 & 0xff)}, {-dmin * (float) (n & 0xff), -dmin * (float) (n >> 8 & 0xff)}};
    }
};

// d, 8 scales of 6 bits (2 above, 4 below), qs[128]: 16 bytes a sub-block of 32;
// w = d (ls - 32) level[q]
template <> struct quant<ZEST_TYPE_IQ4_XS> {
    struct raw { uint4 q; uint2 head; };
    static constexpr int BYTES = 136, CHUNKS = 8;
    static __device__ raw load(const uint8_t * row, int64_t chunk) {
        const uint8_t * p = row + (chunk >> 3) * BYTES;
        return {load_as<uint4>(p + 8 + (chunk & 7) * 16), *reinterpret_cast<const uint2 *>(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][4]) { quant<ZEST_TYPE_IQ4_NL>::codes({r.q, 0}, c); }
    static __device__ half_scales scales(const raw & r, int64_t chunk) {
        const int s = (int) (chunk & 7);
        const int ls = (r.head.y >> 4 * s & 15) | (r.head.x >> (16 + 2 * s) & 3) << 4;
        const float d = half_to_float(r.head.x) * (float) (ls - 32);
        return {{d, d}, {0.0f, 0.0f}};
    }
};

constexpr int GROUPS = 4;        // lane groups of a wave: each takes a chunk of a step
constexpr int CELL = 112;        // bytes of a chunk of one row of x, as prepared: digits, factors, sums
constexpr int LDS_MOST = 160 * 1024;

struct matvec_args {
    const float * x;
    int64_t ldx, row_bytes;
    int32_t M, chunks, glu;      // chunks of a row; glu: the kind, -1: none
    const uint8_t * w[MAX_N];
    const float * res[MAX_N];
    float * y[MAX_N];
    int64_t ldy[MAX_N], ldr[MAX_N];
    int32_t N[MAX_N], tiles[MAX_N];  // tiles: of the weights up to this one
    int32_t n, all_tiles;
    int32_t wk, wr;              // waves that share a tile's chunks, tiles of a workgroup
    int32_t seg_steps, segs;     // steps of a segment of K, segments
    uint8_t * cells;             // prepared by prepare_kernel, [chunk][row]
};

// x as whole numbers: of every 32 consecutive values (whose largest magnitude lies
// in [2^e, 2^(e+1))) v = rint(x 2^(21-e)), |v| < 2^22, cut in three signed bytes v =
// d0 2^16 + d1 2^8 + d2. So products with the weights' codes are exact, in 32 bits,
// and a row of x is met to 2^-22 of the largest of its 32. A cell: [half][digit][16
// bytes], the halves' factors 2^(e-21) (NaN where a value is not finite), their sums.
//
// Eight lanes prepare 32 values of a row, four each; the values past 2^-126 of
// nothing (e below -105) count as zeros.
template <int TYPE> __device__ inline void prepare(const float * x, int64_t ldx, int block, int m, int M, int j, uint8_t * cells) {
    const float4 f = *reinterpret_cast<const float4 *>(x + m * ldx + (int64_t) block * 32 + j * 4);
    const float v[4] = {f.x, f.y, f.z, f.w};
    uint32_t e = 22;
#pragma unroll
    for (int i = 0; i < 4; i++) e = max(e, __float_as_uint(v[i]) >> 23 & 0xffu);
    float sum = (v[0] + v[1]) + (v[2] + v[3]);
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) e = max(e, (uint32_t) __shfl_xor((int) e, off));
    sum += __shfl_xor(sum, 1);
    sum += __shfl_xor(sum, 2);
    const bool odd = e == 255;
    const float up = odd ? 0.0f : __uint_as_float((275 - e) << 23), down = odd ? NAN : __uint_as_float((e - 21) << 23);
    uint32_t d[3] = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int q = odd ? 0 : (int) __builtin_rintf(v[i] * up);
        const int d2 = (int8_t) q, q1 = (q - d2) >> 8, d1 = (int8_t) q1, d0 = (q1 - d1) >> 8;
        d[0] |= (uint32_t) (d0 & 255) << 8 * i;
        d[1] |= (uint32_t) (d1 & 255) << 8 * i;
        d[2] |= (uint32_t) (d2 & 255) << 8 * i;
    }
    // the half's place: Q4_K's chunks hold a half each of two sub-blocks
    const int chunk = TYPE == ZEST_TYPE_Q4_K ? (block & ~1) + (j >> 2) : block, half = TYPE == ZEST_TYPE_Q4_K ? block & 1 : j >> 2;
    uint8_t * cell = cells + (int64_t) (chunk * M + m) * CELL;
#pragma unroll
    for (int i = 0; i < 3; i++) *reinterpret_cast<uint32_t *>(cell + half * 48 + i * 16 + (j & 3) * 4) = d[i];
    if ((j & 3) == 0) {
        *reinterpret_cast<float *>(cell + 96 + half * 4) = down;
        *reinterpret_cast<float *>(cell + 104 + half * 4) = sum;
    }
}

template <int TYPE> __global__ __launch_bounds__(256) void prepare_kernel(matvec_args a) {
    const int i = (blockIdx.x * 256 + threadIdx.x) >> 3, m = blockIdx.y;
    if (i < a.chunks) prepare<TYPE>(a.x, a.ldx, i, m, a.M, threadIdx.x & 7, a.cells);
}

// The rows of a tile: of a weight, or of a GLU's gate and up.
struct tile_rows {
    int32_t weight, row0;
};
__device__ inline tile_rows tile_of(const matvec_args & a, int tile) {
    int i = 0;
    while (i < a.n - 1 && tile >= a.tiles[i]) i++;
    return {i, (tile - (i ? a.tiles[i - 1] : 0)) * 16};
}

// A tile is 16 rows of a weight (S = 2: of a GLU's two), a step four chunks of them:
// a lane loads one chunk of one row, 16 bytes of codes (lane l: row l % 16, chunk l /
// 16), and v_mfma_i32_16x16x64_i8 multiplies each lane's 16 codes of a half with the
// three digits of a row of x for its own chunk: the first operand's row 4 b + i is
// digit i of lane group b's chunk, and zero for the other groups' places, so that
// lane (row, b) of the result holds its own chunk's three sums in its first three
// registers. Scales are then one value a lane, and a chunk costs a lane a conversion
// and a few fused products for a row of x.
//
// HBM bound: a weight's bytes once. The waves of a tile (a.wk of them) share out its
// steps and are joined in shared memory; BLOCK steps of a wave are in flight while it
// computes the last BLOCK.
template <int TYPE, int T, int S, bool COPY> __global__ __launch_bounds__(1024) void matvec_kernel(matvec_args a) {
    typedef quant<TYPE> Q;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    constexpr int BLOCK = S == 2 ? 2 : 4;
    constexpr bool ONE_SCALE = TYPE != ZEST_TYPE_Q4_K, OFFSETS = TYPE == ZEST_TYPE_Q4_K || TYPE == ZEST_TYPE_Q4_1;
    extern __shared__ __align__(16) uint8_t sh[];
    // sh: 16 zeros, the cells of a segment, the waves' results
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4, col = lane & 15;
    const int wr = wave / a.wk, wk = wave - wr * a.wk;
    const int M = a.M, steps = (a.chunks + GROUPS - 1) / GROUPS, segs = COPY ? a.segs : 1, seg_steps = COPY ? a.seg_steps : steps;
    uint8_t * const cells = sh + 16;
    float * const red = reinterpret_cast<float *>(cells + (int64_t) min(seg_steps * GROUPS, a.chunks) * M * CELL);
    const int wg_tiles = (a.all_tiles + a.wr - 1) / a.wr, rounds = (wg_tiles - (int) blockIdx.x + gridDim.x - 1) / gridDim.x;

    struct place {
        int round, seg, first;  // of a block of this wave's steps
    };
    // steps of segment s that are this wave's: s * seg_steps + wk + i * a.wk
    auto count = [&](int seg) { return max(0, (min(seg_steps, steps - seg * seg_steps) - wk + a.wk - 1) / a.wk); };
    auto rows_of = [&](int round) { return ((int) blockIdx.x + round * (int) gridDim.x) * a.wr + wr; };
    auto next = [&](place p) {
        p.first += BLOCK;
        if (p.first >= count(p.seg)) {
            p.first = 0;
            if (++p.seg == segs) {
                p.seg = 0;
                p.round++;
            }
        }
        return p;
    };
    auto load = [&](typename Q::raw (&buf)[BLOCK][S], place p) {
        if (p.round >= rounds) return;
        const int tile = rows_of(p.round);
        if (tile >= a.all_tiles) return;
        const tile_rows t = tile_of(a, tile);
        const int row = min(t.row0 + col, a.N[t.weight] - 1), n = count(p.seg);
        const uint8_t * at[S];
#pragma unroll
        for (int s = 0; s < S; s++) at[s] = a.w[S == 2 ? s : t.weight] + row * a.row_bytes;
#pragma unroll
        for (int i = 0; i < BLOCK; i++) {
            if (p.first + i >= n) continue;
            const int chunk = min((p.seg * seg_steps + wk + (p.first + i) * a.wk) * GROUPS + group, a.chunks - 1);
#pragma unroll
            for (int s = 0; s < S; s++) buf[i][s] = Q::load(at[s], chunk);
        }
    };

    float acc[T][S];
    auto clear = [&]() {
#pragma unroll
        for (int m = 0; m < T; m++)
#pragma unroll
            for (int s = 0; s < S; s++) acc[m][s] = 0.0f;
    };
    // this lane's part of the first operand: digit col % 4 of its group's chunk, if its
    // row is the group's, else zeros
    const bool digit = (col >> 2) == group && (col & 3) < 3;
    auto compute = [&](const typename Q::raw (&buf)[BLOCK][S], place p) {
        const int n = count(p.seg);
#pragma unroll
        for (int i = 0; i < BLOCK; i++) {
            if (p.first + i >= n) continue;
            const int step = wk + (p.first + i) * a.wk, chunk = (p.seg * seg_steps + step) * GROUPS + group;
            const bool in = chunk < a.chunks;
            const int local = step * GROUPS + (in ? group : 0);
            i32x4 code[S][2];
            half_scales sc[S];
#pragma unroll
            for (int s = 0; s < S; s++) {
                uint32_t c[2][4];
                Q::codes(buf[i][s], c);
#pragma unroll
                for (int h = 0; h < 2; h++) code[s][h] = i32x4{(int) c[h][0], (int) c[h][1], (int) c[h][2], (int) c[h][3]};
                sc[s] = Q::scales(buf[i][s], min(chunk, a.chunks - 1));
                if (!in) sc[s] = half_scales{{0.0f, 0.0f}, {0.0f, 0.0f}};
            }
            const uint8_t * cell = cells + local * M * CELL;
            const uint8_t * from = digit && in ? cell + (col & 3) * 16 : sh;
            const int stride = digit && in ? CELL : 0, half_at = digit && in ? 48 : 0;
#pragma unroll
            for (int m = 0; m < T; m++) {
                if (m >= M) continue;
                const i32x4 x0 = *reinterpret_cast<const i32x4 *>(from + m * stride), x1 = *reinterpret_cast<const i32x4 *>(from + m * stride + half_at);
                const float4 f = *reinterpret_cast<const float4 *>(cell + m * CELL + 96);  // the halves' factors and sums
#pragma unroll
                for (int s = 0; s < S; s++) {
                    auto number = [](i32x4 d) { return fmaf((float) d[0], 65536.0f, (float) ((d[1] << 8) + d[2])); };
                    i32x4 d = __builtin_amdgcn_mfma_i32_16x16x64_i8(x0, code[s][0], i32x4{}, 0, 0, 0);
                    if constexpr (ONE_SCALE) {
                        d = __builtin_amdgcn_mfma_i32_16x16x64_i8(x1, code[s][1], d, 0, 0, 0);
                        acc[m][s] = fmaf(number(d), sc[s].scale[0] * f.x, acc[m][s]);
                        if constexpr (OFFSETS) acc[m][s] = fmaf(f.z + f.w, sc[s].offset[0], acc[m][s]);
                    } else {
                        const i32x4 e = __builtin_amdgcn_mfma_i32_16x16x64_i8(x1, code[s][1], i32x4{}, 0, 0, 0);
                        acc[m][s] = fmaf(number(d), sc[s].scale[0] * f.x, acc[m][s]);
                        acc[m][s] = fmaf(number(e), sc[s].scale[1] * f.y, acc[m][s]);
                        acc[m][s] = fmaf(f.z, sc[s].offset[0], acc[m][s]);
                        acc[m][s] = fmaf(f.w, sc[s].offset[1], acc[m][s]);
                    }
                }
            }
        }
    };
    // the cells of a segment, in shared memory
    auto fill = [&](int seg) {
        if (threadIdx.x < 4) reinterpret_cast<uint32_t *>(sh)[threadIdx.x] = 0;
        if constexpr (COPY) {
            const int first = seg * seg_steps * GROUPS, n = min(seg_steps * GROUPS, a.chunks - first) * M * (CELL / 16);
            const uint4 * from = reinterpret_cast<const uint4 *>(a.cells + (int64_t) first * M * CELL);
            for (int i = threadIdx.x; i < n; i += blockDim.x) reinterpret_cast<uint4 *>(cells)[i] = from[i];
        } else {
            const int lanes = a.chunks * 8;
            for (int i = threadIdx.x; i < lanes; i += blockDim.x)
                for (int m = 0; m < M; m++) prepare<TYPE>(a.x, a.ldx, i >> 3, m, M, i & 7, cells);
        }
        __syncthreads();
    };
    // the waves' sums of a round's tiles: of the lane groups, then of the waves
    auto finish = [&](int round) {
        float * const mine = red + wave * T * S * 16;
#pragma unroll
        for (int m = 0; m < T; m++) {
            if (m >= M) continue;
#pragma unroll
            for (int s = 0; s < S; s++) {
                float v = acc[m][s];
                v += __shfl_xor(v, 16);
                v += __shfl_xor(v, 32);
                if (group == 0) mine[(m * S + s) * 16 + col] = v;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.wr * M * 16; i += blockDim.x) {
            const int c = i & 15, m = (i >> 4) % M, r = (i >> 4) / M, tile = ((int) blockIdx.x + round * (int) gridDim.x) * a.wr + r;
            if (tile >= a.all_tiles) continue;
            const tile_rows t = tile_of(a, tile);
            const int row = t.row0 + c;
            if (row >= a.N[t.weight]) continue;
            float v[S];
#pragma unroll
            for (int s = 0; s < S; s++) {
                v[s] = 0.0f;
                for (int w = 0; w < a.wk; w++) v[s] += red[((r * a.wk + w) * T * S + m * S + s) * 16 + c];
            }
            float out = S == 2 ? zest::glu(a.glu, v[0], v[S - 1]) : v[0];
            if (a.res[t.weight]) out += a.res[t.weight][m * a.ldr[t.weight] + row];
            a.y[t.weight][m * a.ldy[t.weight] + row] = out;
        }
        __syncthreads();
    };
    // one block: the next one requested, this one computed; what follows it
    auto turn = [&](typename Q::raw (&now)[BLOCK][S], typename Q::raw (&then)[BLOCK][S], place p) {
        const place q = next(p);
        if (p.first == 0) {
            if (p.seg == 0) clear();
            if (segs > 1 || p.round == 0) {
                if (segs > 1) __syncthreads();
                fill(p.seg);
            }
        }
        load(then, q);
        if (rows_of(p.round) < a.all_tiles) compute(now, p);
        if (q.round != p.round) finish(p.round);
        return q;
    };
    typename Q::raw one[BLOCK][S], two[BLOCK][S];
    place p{0, 0, 0};
    load(one, p);
    while (p.round < rounds) {
        p = turn(one, two, p);
        if (p.round < rounds) p = turn(two, one, p);
    }
}

// ---- the host's plan ----------------------------------------------------------------

struct matvec_plan {
    int wk, wr, workgroups, seg_steps, segs;
    bool copy;        // x is prepared by a kernel of its own
    size_t lds, bytes;
};

matvec_plan plan_of(int64_t M, int64_t K, int n, const int64_t * N, bool glu) {
    matvec_plan p{};
    const int chunks = (int) (K / 32), steps = (chunks + GROUPS - 1) / GROUPS, T = M <= 4 ? 4 : M <= 8 ? 8 : 16, S = glu ? 2 : 1;
    int64_t tiles = 0;
    for (int i = 0; i < (glu ? 1 : n); i++) tiles += (N[i] + 15) / 16;
    p.wr = tiles <= 2 * 256 ? 1 : tiles <= 8 * 256 ? 2 : 4;
    const int most = p.wr == 1 && tiles > 256 ? 8 : 16 / p.wr;
    p.wk = 1;
    for (int w = 1; w <= most; w++)
        if ((steps + w - 1) / w < (steps + p.wk - 1) / p.wk) p.wk = w;
    const size_t red = (size_t) p.wk * p.wr * T * S * 16 * 4, room = LDS_MOST - 16 - red;
    p.seg_steps = (int) std::min<size_t>(steps, room / ((size_t) GROUPS * M * CELL));
    p.segs = (steps + p.seg_steps - 1) / p.seg_steps;
    p.copy = p.segs > 1 || M > 4;
    p.lds = 16 + (size_t) std::min(p.seg_steps * GROUPS, chunks) * M * CELL + red;
    p.workgroups = (int) std::min<int64_t>((tiles + p.wr - 1) / p.wr, 512);
    if (p.lds > LDS_MOST / 2 || p.wk * p.wr > 8) p.workgroups = std::min(p.workgroups, 256);
    p.bytes = std::max<size_t>(16, p.copy ? (size_t) chunks * M * CELL : 0);
    return p;
}

bool supported(int type) {
    switch (type) {
        case ZEST_TYPE_Q4_0:
        case ZEST_TYPE_Q4_1:
        case ZEST_TYPE_Q8_0:
        case ZEST_TYPE_Q4_K:
        case ZEST_TYPE_IQ4_NL:
        case ZEST_TYPE_IQ4_XS: return true;
        default: return false;
    }
}

bool aligned(const void * p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Lets a kernel have all of a CU's shared memory, once a device (threads that launch
// it for the first time at once set the same value).
template <auto KERNEL> int allow_lds(const char * me) {
    static std::atomic<uint64_t> set{0};  // a bit a device, those past the 64th every time
    int device = 0;
    if (const hipError_t e = hipGetDevice(&device); e != hipSuccess) return zest::fail(ZEST_E_HIP, "%s: current device: %s", me, hipGetErrorString(e));
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (set.load(std::memory_order_acquire) & bit) return ZEST_OK;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, LDS_MOST);
    if (e != hipSuccess) return zest::fail(ZEST_E_HIP, "%s: shared memory attribute: %s", me, hipGetErrorString(e));
    set.fetch_or(bit, std::memory_order_release);
    return ZEST_OK;
}

template <int TYPE, int T, int S, bool COPY> int launch(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (const int st = allow_lds<&matvec_kernel<TYPE, T, S, COPY>>(me)) return st;
    if (COPY) hipLaunchKernelGGL(prepare_kernel<TYPE>, dim3((unsigned) ((a.chunks * 8 + 255) / 256), (unsigned) a.M), dim3(256), 0, s, a);
    hipLaunchKernelGGL((matvec_kernel<TYPE, T, S, COPY>), dim3((unsigned) p.workgroups), dim3((unsigned) (p.wk * p.wr * 64)), p.lds, s, a);
    return zest::check_launch(me);
}

template <int TYPE, int S> int launch(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (a.M > 8) return launch<TYPE, 16, S, true>(a, p, s, me);
    if (a.M > 4) return launch<TYPE, 8, S, true>(a, p, s, me);
    if (p.copy) return launch<TYPE, 4, S, true>(a, p, s, me);
    if (a.M > 2) return launch<TYPE, 4, S, false>(a, p, s, me);
    return a.M > 1 ? launch<TYPE, 2, S, false>(a, p, s, me) : launch<TYPE, 1, S, false>(a, p, s, me);
}

template <int TYPE> int launch(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    return a.glu >= 0 ? launch<TYPE, 2>(a, p, s, me) : launch<TYPE, 1>(a, p, s, me);
}

int launch(int type, const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    switch (type) {
        case ZEST_TYPE_Q4_0: return launch<ZEST_TYPE_Q4_0>(a, p, s, me);
        case ZEST_TYPE_Q4_1: return launch<ZEST_TYPE_Q4_1>(a, p, s, me);
        case ZEST_TYPE_Q8_0: return launch<ZEST_TYPE_Q8_0>(a, p, s, me);
        case ZEST_TYPE_Q4_K: return launch<ZEST_TYPE_Q4_K>(a, p, s, me);
        case ZEST_TYPE_IQ4_NL: return launch<ZEST_TYPE_IQ4_NL>(a, p, s, me);
        default: return launch<ZEST_TYPE_IQ4_XS>(a, p, s, me);
    }
}

// The checks and the launch of both entry points; glu: the kind, -1: none.
int matvec(const char * me, int glu, int type, const float * x, int64_t M, int64_t K, int64_t ldx, int n, const void * const * w,
           const int64_t * N, const float * const * res, const int64_t * ldr, float * const * y, const int64_t * ldy,
           void * workspace, size_t workspace_bytes, void * stream) {
    if (!supported(type)) return zest::fail(ZEST_E_UNSUPPORTED, "%s: no kernel for weight type %d", me, type);
    ZEST_REQUIRE(M > 0 && M <= MAX_M, "%s: %lld rows of x (1..%d)", me, (long long) M, MAX_M);
    const size_t row_bytes = K > 0 && K <= (1 << 20) ? zest_raw_row_bytes(type, K) : 0;
    ZEST_REQUIRE(row_bytes > 0, "%s: K=%lld (a multiple of type %d's block up to 2^20)", me, (long long) K, type);
    ZEST_REQUIRE(x && aligned(x, 16) && (M == 1 || (ldx >= K && ldx % 4 == 0 && ldx < (1ll << 31))), "%s: rows of x 16-byte aligned, at least K=%lld apart: ldx=%lld", me,
                 (long long) K, (long long) ldx);
    const int outs = glu >= 0 ? 1 : n;
    matvec_args a{};
    a.x = x;
    a.ldx = M == 1 ? K : ldx;
    a.row_bytes = (int64_t) row_bytes;
    a.M = (int32_t) M;
    a.chunks = (int32_t) (K / 32);
    a.n = outs;
    a.glu = glu;
    int64_t tiles = 0;
    for (int i = 0; i < n; i++) {
        ZEST_REQUIRE(w[i] && aligned(w[i], row_align(type)), "%s: weight %d: rows %d-byte aligned wanted", me, i, row_align(type));
        ZEST_REQUIRE(N[i] > 0 && N[i] <= (1 << 26), "%s: weight %d: N=%lld", me, i, (long long) N[i]);
        a.w[i] = (const uint8_t *) w[i];
        a.N[i] = (int32_t) N[i];
        if (i < outs) tiles += (N[i] + 15) / 16;
        a.tiles[i] = (int32_t) tiles;
    }
    for (int i = 0; i < outs; i++) {
        ZEST_REQUIRE(y[i] && aligned(y[i], 4) && (M == 1 || (ldy[i] >= N[i] && ldy[i] < (1ll << 31))), "%s: output %d: ldy=%lld for N=%lld", me, i, (long long) (M == 1 ? 0 : ldy[i]),
                     (long long) N[i]);
        a.y[i] = y[i];
        a.ldy[i] = M == 1 ? N[i] : ldy[i];
        if (res && res[i]) {
            ZEST_REQUIRE(aligned(res[i], 4) && (M == 1 || (ldr && ldr[i] >= N[i] && ldr[i] < (1ll << 31))), "%s: residual %d", me, i);
            a.res[i] = res[i];
            a.ldr[i] = M == 1 ? N[i] : ldr[i];
        }
    }
    for (int i = 0; i < outs; i++) {
        const size_t ldo = (size_t) a.ldy[i] * 4, width = (size_t) N[i] * 4;
        ZEST_REQUIRE(zest::kv_rows_apart(x, a.ldx * 4, K * 4, y[i], ldo, width, M), "%s: output %d overlaps x", me, i);
        for (int j = 0; j < n; j++)
            ZEST_REQUIRE(zest::kv_rows_apart(w[j], 0, (size_t) N[j] * row_bytes, y[i], 0, (size_t) (M - 1) * ldo + width, 1),
                         "%s: output %d overlaps weight %d", me, i, j);
        for (int j = 0; j < outs; j++) {
            ZEST_REQUIRE(j <= i || zest::kv_rows_apart(y[j], a.ldy[j] * 4, (size_t) N[j] * 4, y[i], ldo, width, M), "%s: outputs %d and %d overlap", me, i, j);
            ZEST_REQUIRE(!a.res[j] || (j == i && a.res[j] == y[i] && a.ldr[j] == a.ldy[i]) ||
                             zest::kv_rows_apart(a.res[j], a.ldr[j] * 4, (size_t) N[j] * 4, y[i], ldo, width, M),
                         "%s: output %d overlaps residual %d without being it", me, i, j);
        }
    }
    // (a GLU's plan is that of two weights as far as its workspace goes)
    const matvec_plan p = plan_of(M, K, n, N, glu >= 0);
    ZEST_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes, "%s: workspace of %zu bytes, 16-byte aligned, wanted", me, p.bytes);
    a.all_tiles = (int32_t) tiles;
    a.wk = p.wk, a.wr = p.wr, a.seg_steps = p.seg_steps, a.segs = p.segs;
    a.cells = (uint8_t *) workspace;
    return launch(type, a, p, zest::as_stream(stream), me);
}

} // namespace

extern "C" {

size_t zest_matvec_workspace(int type, int64_t M, int64_t K, int n, const int64_t * N) {
    if (!supported(type) || M <= 0 || M > MAX_M || K <= 0 || K > (1 << 20) || n < 1 || n > MAX_N || !N) return 0;
    return std::max<size_t>(16, (size_t) (K / 32) * M * CELL);
}

int zest_matvec(int type, const float * x, int64_t M, int64_t K, int64_t ldx, int n, const void * const * w, const int64_t * N,
                const float * const * res, const int64_t * ldr, float * const * y, const int64_t * ldy, void * workspace,
                size_t workspace_bytes, void * stream) {
    ZEST_REQUIRE(n >= 1 && n <= MAX_N, "zest_matvec: %d weights (1..%d)", n, MAX_N);
    ZEST_REQUIRE(w && N && y && (M == 1 || ldy), "zest_matvec: null pointer");
    return matvec("zest_matvec", -1, type, x, M, K, ldx, n, w, N, res, ldr, y, ldy, workspace, workspace_bytes, stream);
}

int zest_matvec_glu(int kind, int type, const float * x, int64_t M, int64_t K, int64_t ldx, const void * gate, const void * up, int64_t F,
                    float * y, int64_t ldy, void * workspace, size_t workspace_bytes, void * stream) {
    if (kind < ZEST_GLU_REGLU || kind > ZEST_GLU_GEGLU_QUICK) return zest::fail(ZEST_E_UNSUPPORTED, "zest_matvec_glu: GLU kind %d", kind);
    const void * const w[2] = {gate, up};
    const int64_t N[2] = {F, F};
    return matvec("zest_matvec_glu", kind, type, x, M, K, ldx, 2, w, N, nullptr, nullptr, &y, &ldy, workspace, workspace_bytes, stream);
}

} // extern "C"

// Products of a few rows with GGUF weights as they are (include/zest/decode.h):
// y[m][n] = sum_k x[m][k] W[n][k], HBM bound by the weights' bytes.
//
// A chunk is what a lane loads of a weight row at a time: 32 values, of Q4_K 64. Its
// codes, signed bytes, come in parts of 16; two parts are a block of 32 consecutive
// values, w = code * scale + offset.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_device.h"
#include "zest/decode.h"
#include "zest_common.h"
#include "zest_device.h"

namespace {

constexpr int MAX_M = ZEST_MATVEC_MAX_ROWS, MAX_N = ZEST_MATVEC_MAX_GROUP;

__device__ inline float half_to_float(uint32_t h) { return (float) __builtin_bit_cast(_Float16, (uint16_t) h); }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ inline uint4 as_uint4(u32x4 v) { return make_uint4(v.x, v.y, v.z, v.w); }

// Words of a row, which need not be aligned to the load (the hardware takes any). By a
// pointer to global memory: a load by a generic one is waited for with all others.
typedef const __attribute__((address_space(1))) uint8_t * bytes_t;
__device__ inline uint4 load_words4(bytes_t p) {
    typedef u32x4 any __attribute__((aligned(2)));
    return as_uint4(*(const __attribute__((address_space(1))) any *) p);
}
__device__ inline uint2 load_words2(bytes_t p) {
    typedef u32x2 any __attribute__((aligned(2)));
    const u32x2 v = *(const __attribute__((address_space(1))) any *) p;
    return make_uint2(v.x, v.y);
}
__device__ inline uint32_t load_word(bytes_t p) {
    typedef uint32_t any __attribute__((aligned(2)));
    return *(const __attribute__((address_space(1))) any *) p;
}
__device__ inline uint32_t load_half(bytes_t p) { return *(const __attribute__((address_space(1))) uint16_t *) p; }

// The published levels of IQ4_NL and IQ4_XS, for the low or the high nibbles of four
// bytes: two byte permutes look up the low and the high eight, and a mask that a
// permute makes of the codes' top bits (it can spread the sign of every other byte)
// picks.
__device__ inline uint32_t iq4_levels(uint32_t n, bool high) {
    constexpr auto four = [](int x, int y, int z, int w) { return (uint32_t) (x & 255) | (uint32_t) (y & 255) << 8 | (uint32_t) (z & 255) << 16 | (uint32_t) (w & 255) << 24; };
    constexpr uint32_t T0 = four(-127, -104, -83, -65), T1 = four(-49, -35, -22, -10), T2 = four(1, 13, 25, 38), T3 = four(53, 69, 89, 113);
    const uint32_t sel = (high ? n >> 4 : n) & 0x07070707u, top = high ? n : n << 4;  // top bits in bit 7
    const uint32_t m = __builtin_amdgcn_perm(top << 8, top, 0x090b080au);
    return (__builtin_amdgcn_perm(T3, T2, sel) & m) | (__builtin_amdgcn_perm(T1, T0, sel) & ~m);
}

constexpr int row_align(int type) {
    return type == ZEST_TYPE_Q4_K ? 16 : type == ZEST_TYPE_IQ4_XS ? 8 : type == ZEST_TYPE_Q4_1 ? 4 : 2;
}

// Four nibbles less 8, as signed bytes (no byte carries into the next).
__device__ inline uint32_t less_8(uint32_t n) { return ((n & 0x0f0f0f0fu) + 0x78787878u) ^ 0x80808080u; }

// Of a type: blocks of a chunk, whether codes are nibbles less 8 (-8..7), whether
// there are offsets; a chunk's loads, codes and scales.
template <int TYPE> struct quant;

template <int BLOCKS> struct block_scales {
    float scale[BLOCKS], offset[BLOCKS];
};

__device__ inline void words(const uint4 & q, uint32_t w[4]) {
    w[0] = q.x;
    w[1] = q.y;
    w[2] = q.z;
    w[3] = q.w;
}

// d, qs[16], the low nibbles the first 16 values: w = d (q - 8), or d level[q]
template <int TYPE> struct quant_nibbles {
    struct raw { uint4 q; uint32_t d; };
    static constexpr int BLOCKS = 1;
    static constexpr bool NIBBLES = false, OFFSETS = false;
    static __device__ raw load(bytes_t row, int chunk) {
        const bytes_t p = row + chunk * 18;
        return {load_words4(p + 2), load_half(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[1][2][4]) {
        uint32_t w[4];
        words(r.q, w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (TYPE == ZEST_TYPE_Q4_0) {
                const uint32_t s = w[i] ^ 0x88888888u;  // 16 (q - 8), the nibble as a byte's high half
                c[0][0][i] = s << 4 & 0xf0f0f0f0u;
                c[0][1][i] = s & 0xf0f0f0f0u;
            } else {
                c[0][0][i] = iq4_levels(w[i], false);
                c[0][1][i] = iq4_levels(w[i], true);
            }
        }
    }
    static constexpr int WORDS = 4;
    static __device__ void packed(const raw & r, uint32_t w[1][4]) { words(r.q, w[0]); }
    static __device__ void eight(const uint32_t w[1][4], int chunk, int, uint32_t & low, uint32_t & high) {
        if constexpr (TYPE == ZEST_TYPE_Q4_0) {
            const uint32_t s = w[0][chunk] ^ 0x88888888u;
            low = s << 4 & 0xf0f0f0f0u, high = s & 0xf0f0f0f0u;
        } else {
            low = iq4_levels(w[0][chunk], false), high = iq4_levels(w[0][chunk], true);
        }
    }
    static __device__ block_scales<1> scales(const raw & r, int) { return {{half_to_float(r.d) * (TYPE == ZEST_TYPE_Q4_0 ? 0.0625f : 1.0f)}, {0.0f}}; }
};
template <> struct quant<ZEST_TYPE_Q4_0> : quant_nibbles<ZEST_TYPE_Q4_0> {};
template <> struct quant<ZEST_TYPE_IQ4_NL> : quant_nibbles<ZEST_TYPE_IQ4_NL> {};

// d, m, qs[16]: w = d q + m = d (q - 8) + (m + 8 d)
template <> struct quant<ZEST_TYPE_Q4_1> {
    struct raw { uint4 q; uint32_t dm; };
    static constexpr int BLOCKS = 1;
    static constexpr bool NIBBLES = true, OFFSETS = true;
    static __device__ raw load(bytes_t row, int chunk) {
        const bytes_t p = row + chunk * 20;
        return {load_words4(p + 4), load_word(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[1][2][4]) {
        uint32_t w[4];
        words(r.q, w);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            c[0][0][i] = less_8(w[i]);
            c[0][1][i] = less_8(w[i] >> 4);
        }
    }
    static constexpr int WORDS = 4;
    static __device__ void packed(const raw & r, uint32_t w[1][4]) { words(r.q, w[0]); }
    static __device__ void eight(const uint32_t w[1][4], int chunk, int, uint32_t & low, uint32_t & high) {
        low = less_8(w[0][chunk]), high = less_8(w[0][chunk] >> 4);
    }
    static __device__ block_scales<1> scales(const raw & r, int) {
        const float d = half_to_float(r.dm);
        return {{d}, {fmaf(8.0f, d, half_to_float(r.dm >> 16))}};
    }
};

// d, qs[32]: w = d q
template <> struct quant<ZEST_TYPE_Q8_0> {
    struct raw { uint4 q[2]; uint32_t d; };
    static constexpr int BLOCKS = 1;
    static constexpr bool NIBBLES = false, OFFSETS = false;
    static __device__ raw load(bytes_t row, int chunk) {
        const bytes_t p = row + chunk * 34;
        return {{load_words4(p + 2), load_words4(p + 18)}, load_half(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[1][2][4]) {
        words(r.q[0], c[0][0]);
        words(r.q[1], c[0][1]);
    }
    static constexpr int WORDS = 8;
    static __device__ void packed(const raw & r, uint32_t w[2][4]) {
        words(r.q[0], w[0]);
        words(r.q[1], w[1]);
    }
    static __device__ void eight(const uint32_t w[2][4], int chunk, int, uint32_t & low, uint32_t & high) { low = w[0][chunk], high = w[1][chunk]; }
    static __device__ block_scales<1> scales(const raw & r, int) { return {{half_to_float(r.d)}, {0.0f}}; }
};

// d, dmin, 12 bytes of 6-bit scales and minima of 8 blocks of 32, qs[128]: a chunk's
// 64 values in 32 bytes, block 2r in the low nibbles, 2r + 1 in the high ones;
// w = d sc q - dmin m, taken about q = 8 too: the codes' products are then no larger than the
// sum they make, and the offsets of weights that were quantised evenly about 0 all but vanish
template <> struct quant<ZEST_TYPE_Q4_K> {
    struct raw { uint4 q[2], head; };
    static constexpr int BLOCKS = 2;
    static constexpr bool NIBBLES = true, OFFSETS = true;
    static __device__ raw load(bytes_t row, int chunk) {
        const bytes_t p = row + (chunk >> 2) * 144;
        const bytes_t q = p + 16 + (chunk & 3) * 32;
        return {{load_words4(q), load_words4(q + 16)}, load_words4(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[2][2][4]) {
#pragma unroll
        for (int part = 0; part < 2; part++) {
            uint32_t w[4];
            words(r.q[part], w);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                c[0][part][i] = less_8(w[i]);
                c[1][part][i] = less_8(w[i] >> 4);
            }
        }
    }
    static constexpr int WORDS = 8;
    static __device__ void packed(const raw & r, uint32_t w[2][4]) {
        words(r.q[0], w[0]);
        words(r.q[1], w[1]);
    }
    static __device__ void eight(const uint32_t w[2][4], int chunk, int block, uint32_t & low, uint32_t & high) {
        low = less_8(w[0][chunk] >> 4 * block), high = less_8(w[1][chunk] >> 4 * block);
    }
    static __device__ block_scales<2> scales(const raw & r, int chunk) {
        const float d = half_to_float(r.head.x), dmin = half_to_float(r.head.x >> 16);
        // the first four blocks' fields are low 6 bits, the others' 4 bits and the first's top two
        const bool far = chunk & 2;
        const uint32_t a = far ? r.head.y >> 2 & 0x30303030u : r.head.y & 0x3f3f3f3fu, b = far ? r.head.z >> 2 & 0x30303030u : r.head.z & 0x3f3f3f3fu;
        const uint32_t both = far ? r.head.w : 0u;
        const int by = 16 * (chunk & 1);
        const uint32_t s = ((both & 0x0f0f0f0fu) | a) >> by, n = ((both >> 4 & 0x0f0f0f0fu) | b) >> by;
        const float d0 = d * (float) (s & 0xff), d1 = d * (float) (s >> 8 & 0xff);
        return {{d0, d1}, {fmaf(-dmin, (float) (n & 0xff), 8.0f * d0), fmaf(-dmin, (float) (n >> 8 & 0xff), 8.0f * d1)}};
    }
};

// d, 8 scales of 6 bits (2 above, 4 below), qs[128]: 16 bytes a block of 32;
// w = d (ls - 32) level[q]
template <> struct quant<ZEST_TYPE_IQ4_XS> {
    struct raw { uint4 q; uint2 head; };
    static constexpr int BLOCKS = 1;
    static constexpr bool NIBBLES = false, OFFSETS = false;
    static __device__ raw load(bytes_t row, int chunk) {
        const bytes_t p = row + (chunk >> 3) * 136;
        return {load_words4(p + 8 + (chunk & 7) * 16), load_words2(p)};
    }
    static __device__ void codes(const raw & r, uint32_t c[1][2][4]) { quant<ZEST_TYPE_IQ4_NL>::codes({r.q, 0}, c); }
    static constexpr int WORDS = 4;
    static __device__ void packed(const raw & r, uint32_t w[1][4]) { words(r.q, w[0]); }
    static __device__ void eight(const uint32_t w[1][4], int chunk, int, uint32_t & low, uint32_t & high) { quant<ZEST_TYPE_IQ4_NL>::eight(w, chunk, 0, low, high); }
    static __device__ block_scales<1> scales(const raw & r, int chunk) {
        const int s = chunk & 7, ls = (r.head.y >> 4 * s & 15) | (r.head.x >> (16 + 2 * s) & 3) << 4;
        return {{half_to_float(r.head.x) * (float) (ls - 32)}, {0.0f}};
    }
};

constexpr int GROUPS = 4;        // lane groups of a wave: each takes a chunk of a step
constexpr int CELL = 112;        // bytes of 32 values of a row of x, as prepared: digits, factor, sum
constexpr int LDS_MOST = 160 * 1024;

struct matvec_args {
    const float * x;
    int64_t ldx, row_bytes;
    int32_t M, blocks, chunks, glu;  // blocks and chunks of a row; glu: the kind, -1: none
    const uint8_t * w[MAX_N];
    const float * res[MAX_N];
    float * y[MAX_N];
    int64_t ldy[MAX_N], ldr[MAX_N];
    int32_t N[MAX_N], tiles[MAX_N];  // tiles: of the weights up to this one
    int32_t n, all_tiles;
    int32_t wk, wr;              // waves that share a tile's chunks, tiles of a workgroup
    int32_t seg_steps, segs;     // steps of a segment of K, segments
    uint8_t * cells;             // prepared by prepare_kernel, [block][row]
    int32_t rows[MAX_N];         // rows: of the weights up to this one
    int32_t pieces, each, more;  // pieces of a row; rows of a stream's workgroup
};

// Another lane's value: 0xb1 and 0x4e swap lanes and pairs of a quad, 0x141 mirrors eight.
template <int CTRL> __device__ inline float dpp(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, false)); }

// The sum of a value over the four lane groups of 16.
__device__ inline float over_groups(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(h[0]) + __uint_as_float(h[1]);
}

// x as whole numbers: of every 32 consecutive values (whose largest magnitude is below
// 2^(e+1) (1 - 2^-8 - 2^-15): the last 2^-8 counts to the next e) v = rint(x 2^(22-e)), cut
// in three signed bytes v = d0 2^16 + d1 2^8 + d2, |d0| <= 127. So products with the
// weights' codes are exact, in 32 bits, and a row of x is met to 2^-22 of the largest of its
// 32 (2^-23 and a little). A cell: [part][digit][16 bytes], the factor 2^(e-22) (NaN where a
// value is not finite), the values' sum.
//
// Eight lanes prepare a block of a row, four values each: the four digits of each kind,
// the factor and the sum. Where e is below -104 (the last bit below 2^-126), it counts
// as -104.
struct prepared {
    uint32_t digits[3];
    float factor, sum;
};
__device__ inline prepared prepare(float4 f) {
    const float v[4] = {f.x, f.y, f.z, f.w};
    uint32_t e = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) e = max(e, __float_as_uint(v[i]) & 0x7fffffffu);
    prepared r{{0, 0, 0}, 0.0f, (v[0] + v[1]) + (v[2] + v[3])};
    // over the quad, then the other quad of the eight
    e = max(e, (uint32_t) __builtin_amdgcn_mov_dpp((int) e, 0xb1, 0xf, 0xf, false));
    e = max(e, (uint32_t) __builtin_amdgcn_mov_dpp((int) e, 0x4e, 0xf, 0xf, false));
    e = max(e, (uint32_t) __builtin_amdgcn_mov_dpp((int) e, 0x141, 0xf, 0xf, false));
    r.sum += dpp<0xb1>(r.sum);
    r.sum += dpp<0x4e>(r.sum);
    r.sum += dpp<0x141>(r.sum);
    const bool odd = e >= 0x7f800000u;
    e = max((e + 0x10200u) >> 23, 23u);
    const float up = odd ? 0.0f : __uint_as_float((276 - e) << 23);
    r.factor = odd ? NAN : __uint_as_float((e - 22) << 23);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int q = odd ? 0 : (int) __builtin_rintf(v[i] * up);
        const int d2 = (int8_t) q, q1 = (q - d2) >> 8, d1 = (int8_t) q1, d0 = (q1 - d1) >> 8;
        r.digits[0] |= (uint32_t) (d0 & 255) << 8 * i;
        r.digits[1] |= (uint32_t) (d1 & 255) << 8 * i;
        r.digits[2] |= (uint32_t) (d2 & 255) << 8 * i;
    }
    return r;
}

// Cells in global memory: a stream's, of a block and a row, or (of TILE bytes) a tile's, of
// a block for MAX_M rows of x: [digit][lane group][row][8 bytes], the rows' factors, and
// their sums where the type has offsets. A lane group's 8 bytes are the digits of values
// 4g..4g+3 and 16+4g..16+4g+3. (Rows of a tile from M on hold anything; nothing is made of them.)
template <int BYTES> __global__ __launch_bounds__(256) void prepare_kernel(matvec_args a) {
    const int items = a.blocks * a.M * 8, by = gridDim.x * 256;
    for (int i = blockIdx.x * 256 + threadIdx.x; i < items; i += by) {  // (a block's eight lanes go in step)
        const int cell = i >> 3, block = cell / a.M, m = cell - block * a.M, j = i & 7;
        const prepared r = prepare(*reinterpret_cast<const float4 *>(a.x + m * a.ldx + block * 32 + j * 4));
        uint8_t * const to = a.cells + (int64_t) (BYTES == CELL ? cell : block) * BYTES;
#pragma unroll
        for (int d = 0; d < 3; d++) *reinterpret_cast<uint32_t *>(to + (BYTES == CELL ? (j >> 2) * 48 + d * 16 + (j & 3) * 4 : d * 512 + (j & 3) * 128 + m * 8 + (j >> 2) * 4)) = r.digits[d];
        if (j) continue;
        if constexpr (BYTES == CELL) {
            *reinterpret_cast<float2 *>(to + 96) = make_float2(r.factor, r.sum);
        } else {
            *reinterpret_cast<float *>(to + 1536 + m * 4) = r.factor;
            if (BYTES > 1600) *reinterpret_cast<float *>(to + 1600 + m * 4) = r.sum;
        }
    }
}

// Entry i of an argument's list, by selection among scalar registers: an index that
// differs between lanes would be a load of the arguments' memory each time, to which
// the compiler would turn a plain selection back.
template <typename V> __device__ inline V pick(const V (&list)[MAX_N], int i) {
    V v = list[0];
#pragma unroll
    for (int k = 1; k < MAX_N; k++) {
        V one = list[k];
        asm("" : "+s"(one));
        v = i == k ? one : v;
    }
    return v;
}

// A tile: its weight (a GLU's gate and up are one) and its number there.
struct tile_place {
    int32_t weight, number;
};
__device__ inline tile_place tile_of(const matvec_args & a, int tile) {
    int weight = 0, before = 0;
#pragma unroll
    for (int k = 0; k < MAX_N - 1; k++) {
        const bool past = k < a.n - 1 && tile >= a.tiles[k];
        weight = past ? k + 1 : weight;
        before = past ? a.tiles[k] : before;
    }
    return {weight, tile - before};
}

// What becomes of the sums v (S of them, a GLU's gate and up) of a weight's row and row
// m of x.
template <int S> __device__ inline void store_row(const matvec_args & a, int weight, int row, int m, const float v[S]) {
    float out = S == 2 ? zest::glu(a.glu, v[0], v[S - 1]) : v[0];
    typedef __attribute__((address_space(1))) float * global_floats;
    const global_floats res = (global_floats) pick(a.res, weight), y = (global_floats) pick(a.y, weight);
    if (res) out += res[m * pick(a.ldr, weight) + row];
    y[m * pick(a.ldy, weight) + row] = out;
}

// ---- up to 16 rows of x, tile by tile -------------------------------------------------

// What the lanes of a wave wrote to shared memory, which it serves in order, is read after it.
__device__ inline void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int TYPE> constexpr int TILE_CELL = quant<TYPE>::OFFSETS ? 1664 : 1600;
// Words of a weight row's four chunks where they change lanes: codes, scales and offsets, an
// odd number of fours, so that 16 rows' reads spread over all banks; and a wave's bytes, which
// hold its sums afterwards.
template <int TYPE> constexpr int TRADE = (quant<TYPE>::WORDS * 4 + quant<TYPE>::BLOCKS * (quant<TYPE>::OFFSETS ? 8 : 4)) | 4;
template <int TYPE, int H> constexpr int WAVE_BYTES = TRADE<TYPE> * 64 > H * 1024 ? TRADE<TYPE> * 64 : H * 1024;

// A tile is 16 rows of a weight (H = 2: 32, or with S = 2 a GLU's gate and up), a step four
// chunks of them. A lane loads one chunk of one row (lane l: row l / 4, chunk l % 4, so that
// four lanes read consecutive bytes), and the wave trades in its own shared memory: lane (row
// l % 16, group l / 16) gets its eight values of every block, which is what v_mfma_i32_16x16x32_i8 takes of a block of 16 rows,
// and all four scales. Three products, one a digit of x, give
// the 16 rows' sums with all rows of x: a lane has those of its weight row and four rows of
// x, and puts the digits together and to its fp32 sums by scale and factor.
//
// x's cells lie in shared memory, all of K's or a segment's. The waves of a tile (a.wk of
// them) each take a run of its steps; AHEAD steps of a wave are in flight while it computes
// the AHEAD before them (twice as many were slower: 154 us for 115), and the waves' sums are
// joined in shared memory. 151936 rows of 2560 IQ4_XS by 16: 100 us, of which the loads alone
// take 76 and the products alone 82; with products of a lane's own 16 codes, a row of x at a
// time as below, 190.
template <int TYPE, int H, int S> __global__ __launch_bounds__(1024) void matvec_kernel(matvec_args a) {
    typedef quant<TYPE> Q;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    constexpr int B = Q::BLOCKS, AHEAD = 16 / (H * Q::WORDS), ROWS = S == 2 ? 16 : 16 * H, CELLS = TILE_CELL<TYPE>;
    extern __shared__ __align__(16) uint8_t sh[];
    // sh: the cells of a segment, the waves' own
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4, col = lane & 15;
    const int wr = wave / a.wk, wk = wave - wr * a.wk;
    const int steps = (a.chunks + GROUPS - 1) / GROUPS, segs = a.segs, seg_steps = a.seg_steps;
    uint8_t * const own = sh + min(seg_steps * GROUPS, a.chunks) * B * CELLS + wave * WAVE_BYTES<TYPE, H>;
    uint32_t * const to = reinterpret_cast<uint32_t *>(own) + (lane >> 2) * TRADE<TYPE>;
    const uint32_t * const from = reinterpret_cast<const uint32_t *>(own) + col * TRADE<TYPE>;
    const int wg_tiles = (a.all_tiles + a.wr - 1) / a.wr, rounds = (wg_tiles - (int) blockIdx.x + gridDim.x - 1) / gridDim.x;

    // A block of this wave's steps: of round `round` and segment `seg`, from step `at` of
    // the segment on, up to `end`.
    struct place {
        int round, seg, at, end;
    };
    auto start = [&](int round, int seg) {
        const int n = min(seg_steps, steps - seg * seg_steps);
        return place{round, seg, n * wk / a.wk, n * (wk + 1) / a.wk};
    };
    auto next = [&](place p) {
        p.at += AHEAD;
        if (p.at < p.end) return p;
        return p.seg + 1 < segs ? start(p.round, p.seg + 1) : start(p.round + 1, 0);
    };
    auto tile_at = [&](int round) { return ((int) blockIdx.x + round * (int) gridDim.x) * a.wr + wr; };
    auto load = [&](typename Q::raw (&buf)[AHEAD][H], place p) {
        // (every lane loads, whatever there is left to load, so that the loads in flight are known)
        const tile_place t = tile_of(a, min(tile_at(p.round), a.all_tiles - 1));
        const int last = pick(a.N, t.weight) - 1;
        bytes_t at[H];
#pragma unroll
        for (int h = 0; h < H; h++)
            at[h] = (bytes_t) (S == 2 ? a.w[h] : pick(a.w, t.weight)) + (int64_t) min(t.number * ROWS + (S == 2 ? 0 : h * 16) + (lane >> 2), last) * a.row_bytes;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int chunk = min((p.seg * seg_steps + min(p.at + i, max(p.end - 1, 0))) * GROUPS + (lane & 3), a.chunks - 1);
#pragma unroll
            for (int h = 0; h < H; h++) buf[i][h] = Q::load(at[h], chunk);
        }
    };

    float acc[H][4];
    auto clear = [&]() {
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc[h][r] = 0.0f;
    };
    auto compute = [&](const typename Q::raw (&buf)[AHEAD][H], place p) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            if (p.at + i >= p.end) continue;
            const int chunk0 = (p.seg * seg_steps + p.at + i) * GROUPS;  // group 0's
            uint32_t w[H][Q::WORDS / 4][4];
            f32x4 scale[H][B], offset[H][B];
#pragma unroll
            for (int h = 0; h < H; h++) {
                const int c = lane & 3;
                uint32_t mine[Q::WORDS / 4][4];
                Q::packed(buf[i][h], mine);
                // (past the row's end: any bytes, by a scale of 0)
                const bool in = chunk0 + c < a.chunks;
                const block_scales<B> sc = Q::scales(buf[i][h], min(chunk0 + c, a.chunks - 1));
#pragma unroll
                for (int q = 0; q < Q::WORDS / 4; q++) *reinterpret_cast<u32x4 *>(to + q * 16 + c * 4) = u32x4{mine[q][0], mine[q][1], mine[q][2], mine[q][3]};
#pragma unroll
                for (int b = 0; b < B; b++) {
                    to[Q::WORDS * 4 + b * 4 + c] = __float_as_uint(in ? sc.scale[b] : 0.0f);
                    if constexpr (Q::OFFSETS) to[Q::WORDS * 4 + (B + b) * 4 + c] = __float_as_uint(in ? sc.offset[b] : 0.0f);
                }
                wave_sync();
#pragma unroll
                for (int k = 0; k < GROUPS; k++)
#pragma unroll
                    for (int q = 0; q < Q::WORDS / 4; q++) w[h][q][k] = from[q * 16 + k * 4 + group];
#pragma unroll
                for (int b = 0; b < B; b++) {
                    scale[h][b] = *reinterpret_cast<const f32x4 *>(from + Q::WORDS * 4 + b * 4);
                    if constexpr (Q::OFFSETS) offset[h][b] = *reinterpret_cast<const f32x4 *>(from + Q::WORDS * 4 + (B + b) * 4);
                }
                wave_sync();
            }
#pragma unroll
            for (int c = 0; c < GROUPS; c++) {
                const uint8_t * cell = sh + (min(chunk0 + c, a.chunks - 1) - p.seg * seg_steps * GROUPS) * (B * CELLS);
#pragma unroll
                for (int b = 0; b < B; b++) {
                    long x[3];
#pragma unroll
                    for (int d = 0; d < 3; d++) x[d] = *reinterpret_cast<const long *>(cell + b * CELLS + d * 512 + lane * 8);
                    const f32x4 f = *reinterpret_cast<const f32x4 *>(cell + b * CELLS + 1536 + group * 16);
                    f32x4 sum{};
                    if constexpr (Q::OFFSETS) sum = *reinterpret_cast<const f32x4 *>(cell + b * CELLS + 1600 + group * 16);
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        uint32_t low, high;  // the values' first and second half
                        Q::eight(w[h], c, b, low, high);
                        const long code = (long) ((uint64_t) high << 32 | low);
                        i32x4 d[3];
#pragma unroll
                        for (int k = 0; k < 3; k++) d[k] = __builtin_amdgcn_mfma_i32_16x16x32_i8(x[k], code, i32x4{}, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            // (nibbles' sums |d0| <= 127 8 32 and |d1|, |d2| <= 128 8 32 fit in 32 bits together)
                            const float v = Q::NIBBLES ? (float) ((((d[0][r] << 8) + d[1][r]) << 8) + d[2][r]) : fmaf((float) d[0][r], 65536.0f, (float) ((d[1][r] << 8) + d[2][r]));
                            acc[h][r] = fmaf(v, scale[h][b][c] * f[r], acc[h][r]);
                            if constexpr (Q::OFFSETS) acc[h][r] = fmaf(sum[r], offset[h][b][c], acc[h][r]);
                        }
                    }
                }
            }
        }
    };
    // the cells of a segment, in shared memory
    auto fill = [&](int seg) {
        const int first = seg * seg_steps * GROUPS * B, n = min(seg_steps * GROUPS * B, a.blocks - first) * (CELLS / 16);
        const uint4 * from = reinterpret_cast<const uint4 *>(a.cells + (int64_t) first * CELLS);
        constexpr int AT_ONCE = 9;  // requested together
        for (int i0 = threadIdx.x; i0 < n; i0 += AT_ONCE * blockDim.x) {
            uint4 v[AT_ONCE];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++) v[u] = from[min(i0 + u * (int) blockDim.x, n - 1)];
#pragma unroll
            for (int u = 0; u < AT_ONCE; u++)
                if (i0 + u * (int) blockDim.x < n) reinterpret_cast<uint4 *>(sh)[i0 + u * (int) blockDim.x] = v[u];
        }
        __syncthreads();
    };
    // a round's tiles: the waves of each share out its sums
    auto finish = [&](int round) {
        const int tile = tile_at(round);
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) reinterpret_cast<float *>(own)[(h * 4 + r) * 64 + lane] = acc[h][r];
        if (a.wk > 1) __syncthreads();
        else wave_sync();
        if (tile < a.all_tiles) {
            const tile_place t = tile_of(a, tile);
            const int rows = pick(a.N, t.weight);
            const float * sums = reinterpret_cast<const float *>(own - wk * WAVE_BYTES<TYPE, H>);
            for (int i = wk; i < H / S * 4; i += a.wk) {
                float v[S];
#pragma unroll
                for (int s = 0; s < S; s++) {
                    v[s] = 0.0f;
                    for (int k = 0; k < a.wk; k++) v[s] += sums[k * (WAVE_BYTES<TYPE, H> / 4) + (s * 4 + i) * 64 + lane];
                }
                const int row = t.number * ROWS + (i >> 2) * 16 + col, m = group * 4 + (i & 3);
                if (row < rows && m < a.M) store_row<S>(a, t.weight, row, m, v);
            }
        }
        if (a.wk > 1) __syncthreads();
        else wave_sync();
    };
    // one block: the next one requested, this one computed; what follows it
    auto turn = [&](typename Q::raw (&now)[AHEAD][H], typename Q::raw (&then)[AHEAD][H], place p, bool first) {
        const place q = next(p);
        if (first) {  // of a segment
            if (p.seg == 0) clear();
            if (segs > 1 || p.round == 0) {
                if (segs > 1) __syncthreads();
                fill(p.seg);
            }
        }
        load(then, q);
        if (tile_at(p.round) < a.all_tiles) compute(now, p);
        if (q.round != p.round) finish(p.round);
        return q;
    };
    typename Q::raw one[AHEAD][H], two[AHEAD][H];
    place p = start(0, 0);
    bool first = true;
    load(one, p);
    while (p.round < rounds) {
        place q = turn(one, two, p, first);
        first = q.round != p.round || q.seg != p.seg;
        p = q;
        if (p.round >= rounds) break;
        q = turn(two, one, p, first);
        first = q.round != p.round || q.seg != p.seg;
        p = q;
    }
}

// ---- few rows of x: streams through shared memory ---------------------------------------

// What a type's rows look like to a stream: a unit is UNIT bytes of a row, CHUNKS
// chunks (whole blocks of the format; a multiple of GROUPS, so whole steps), and a
// chunk is read from shared memory, where its row may begin at any multiple of the
// row's alignment.
template <int TYPE> struct stream;

// Shared memory by its address: a read through a pointer that the compiler can follow
// to an object waits for all direct loads into that object.
template <typename V> __device__ inline V lds(uint32_t at) { return *(const __attribute__((address_space(3))) V *) (uintptr_t) at; }
template <typename V> __device__ inline void lds(uint32_t at, V v) { *(__attribute__((address_space(3))) V *) (uintptr_t) at = v; }

// A chunk of 2 bytes of scale and N words of codes, at an even address: whole words are
// read from a whole address on, of which the codes come out by a permute, or are words.
template <int N> __device__ inline void read_scaled(uint32_t at, uint32_t codes[N], uint32_t & scale) {
    uint32_t w[N + 1];
#pragma unroll
    for (int i = 0; i <= N; i++) w[i] = lds<uint32_t>((at & ~3u) + 4 * i);
    const bool odd = at & 2;
    const uint32_t sel = odd ? 0x07060504u : 0x05040302u;
#pragma unroll
    for (int i = 0; i < N; i++) codes[i] = __builtin_amdgcn_perm(w[i + 1], w[i], sel);
    scale = odd ? w[0] >> 16 : w[0] & 0xffffu;
}

template <int TYPE> struct stream_nibbles {
    static constexpr int UNIT = 144, CHUNKS = 8;
    static __device__ typename quant<TYPE>::raw read(uint32_t unit, int chunk) {
        uint32_t w[4], d;
        read_scaled<4>(unit + chunk * 18, w, d);
        return {make_uint4(w[0], w[1], w[2], w[3]), d};
    }
};
template <> struct stream<ZEST_TYPE_Q4_0> : stream_nibbles<ZEST_TYPE_Q4_0> {};
template <> struct stream<ZEST_TYPE_IQ4_NL> : stream_nibbles<ZEST_TYPE_IQ4_NL> {};
template <> struct stream<ZEST_TYPE_Q4_1> {
    static constexpr int UNIT = 160, CHUNKS = 8;
    static __device__ quant<ZEST_TYPE_Q4_1>::raw read(uint32_t unit, int chunk) {
        uint32_t w[5];
#pragma unroll
        for (int i = 0; i < 5; i++) w[i] = lds<uint32_t>(unit + chunk * 20 + 4 * i);
        return {make_uint4(w[1], w[2], w[3], w[4]), w[0]};
    }
};
template <> struct stream<ZEST_TYPE_Q8_0> {
    static constexpr int UNIT = 136, CHUNKS = 4;
    static __device__ quant<ZEST_TYPE_Q8_0>::raw read(uint32_t unit, int chunk) {
        uint32_t w[8], d;
        read_scaled<8>(unit + chunk * 34, w, d);
        return {{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])}, d};
    }
};
template <> struct stream<ZEST_TYPE_Q4_K> {
    static constexpr int UNIT = 144, CHUNKS = 4;
    static __device__ quant<ZEST_TYPE_Q4_K>::raw read(uint32_t unit, int chunk) {
        return {{as_uint4(lds<u32x4>(unit + 16 + 32 * chunk)), as_uint4(lds<u32x4>(unit + 32 + 32 * chunk))}, as_uint4(lds<u32x4>(unit))};
    }
};
template <> struct stream<ZEST_TYPE_IQ4_XS> {
    static constexpr int UNIT = 136, CHUNKS = 8;
    static __device__ quant<ZEST_TYPE_IQ4_XS>::raw read(uint32_t unit, int chunk) {
        const u32x2 head = lds<u32x2>(unit), a = lds<u32x2>(unit + 8 + 16 * chunk), b = lds<u32x2>(unit + 16 + 16 * chunk);
        return {make_uint4(a.x, a.y, b.x, b.y), make_uint2(head.x, head.y)};
    }
};

constexpr int STREAM_WAVES = 8;
constexpr int RAW_CELL = 128;  // of 32 values of x where a stream's workgroups prepare them, over the values themselves
// Units of a row in a piece; the 16-byte granules that hold them wherever the row
// begins; their places in shared memory, an odd number, so that 16 rows' reads spread
// over the banks; a piece's loads.
template <int S> constexpr int UNITS = 2 / S;
template <int TYPE, int S> constexpr int GRANULES = (UNITS<S> * stream<TYPE>::UNIT + 16 - row_align(TYPE) + 15) / 16;
template <int TYPE, int S> constexpr int PLACES = GRANULES<TYPE, S> | 1;
template <int TYPE, int S> constexpr int LOADS = (16 * S * PLACES<TYPE, S> + 63) / 64;

typedef __attribute__((address_space(3))) void * lds_ptr_t;
typedef const __attribute__((address_space(1))) void * global_ptr_t;

// The call's rows are shared out evenly over the workgroups, a workgroup's pieces, 16
// rows by 16, over its waves; the first of either take one more where they do not come
// out even.
struct run {
    int each, more;
    __device__ int start(int i) const { return i * each + min(i, more); }
};

// A row of the call: of which weight, and its number there.
struct call_row {
    int weight, row;
};
__device__ inline call_row row_of(const matvec_args & a, int r) {
    int weight = 0, before = 0;
#pragma unroll
    for (int k = 0; k < MAX_N - 1; k++) {
        const bool past = k < a.n - 1 && r >= a.rows[k];
        weight = past ? k + 1 : weight;
        before = past ? a.rows[k] : before;
    }
    return {weight, r - before};
}

// v_mfma_i32_16x16x64_i8 multiplies the 16 codes of a part that each lane holds of its own
// chunk (lane l: row l % 16, chunk l / 16 of a step) with the three digits of a row of x for
// that chunk: the first operand's row 4 b + i is digit i of lane group b's chunk, and zero
// in the other groups' places, so that lane (row, b) of the result holds its own chunk's
// three sums in its first three registers. Scales are then one value a lane, and a block
// costs a lane a conversion and a few fused products for a row of x.
//
// HBM bound: a weight's bytes once. They come not chunk by chunk into registers, where an
// instruction touches 16 lines or more and a line is asked for three times, but as whole
// granules of contiguous bytes straight into shared memory: RING pieces (two units of 16 rows, 4.6 KB) a wave, requested as soon as their place
// is read. A workgroup's last 16 rows are as many as are left of its share: a row that
// is not there is its neighbour again. So all CUs stream whatever the number of rows. A
// GLU's two weights of 17408 rows of 5120 Q4_K by 4 rows: 29 to 32 us, 3.2 to 3.5 TB/s; 2560
// rows of 9728 Q8_0 by one: 10.8, 1024 of 1024 Q4_0 by 3: 6.1 (a chain of x, its digits and
// the weights). Deeper rings with one workgroup a CU: 38 us for the first.
template <int TYPE, int M, int S, int RING, bool READY>
__global__ __launch_bounds__(STREAM_WAVES * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void stream_kernel(matvec_args a) {
    typedef quant<TYPE> Q;
    typedef stream<TYPE> ST;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    constexpr int B = Q::BLOCKS, U = UNITS<S>, G = GRANULES<TYPE, S>, GP = PLACES<TYPE, S>, NL = LOADS<TYPE, S>, ALIGN = row_align(TYPE);
    constexpr int STEPS = U * (ST::CHUNKS / GROUPS);  // of a piece
    constexpr int CELL_AT = READY ? CELL : RAW_CELL;
    extern __shared__ __align__(1024) uint8_t sh[];
    // sh: the rings, the cells, 16 zeros, the waves' results
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = lane >> 4, col = lane & 15;
    const int pieces = a.pieces, row_bytes = (int) a.row_bytes;
    const run all{a.each, a.more};
    const int first_row = all.start(blockIdx.x), end_row = all.start(blockIdx.x + 1), tiles = (end_row - first_row + 15) / 16;
    const int n = tiles * pieces;
    const run waves{n / STREAM_WAVES, n % STREAM_WAVES};
    const int u0 = waves.start(wave), u1 = waves.start(wave + 1);
    const uint32_t base = (uint32_t) (uintptr_t) (lds_ptr_t) sh, ring = base + wave * (RING * NL * 1024), cells = base + STREAM_WAVES * RING * NL * 1024;
    const uint32_t cell_bytes = (uint32_t) (a.blocks * M * CELL_AT + 1023) & ~1023u, zeros = cells + cell_bytes;
    float * const red = reinterpret_cast<float *>(sh + (zeros + 16 - base));

    // x, or its cells, straight into shared memory, before the weights so that it is not
    // waited for behind them (all of these are waits that this kernel counts itself: one
    // of the compiler's would be for everything on its way)
    for (uint32_t at = wave * 1024; at < cell_bytes; at += STREAM_WAVES * 1024) {
        const uint32_t mine_at = at + lane * 16;
        const uint8_t * from = a.cells + min(mine_at, (uint32_t) (a.blocks * M * CELL_AT) - 16);
        if constexpr (!READY) {  // cell c: row c % M's block c / M
            const int cell = min((int) (mine_at / RAW_CELL), a.blocks * M - 1), block = cell / M, m = cell - block * M;
            from = (const uint8_t *) (a.x + m * a.ldx + block * 32 + (lane & 7) * 4);
        }
        __builtin_amdgcn_global_load_lds((global_ptr_t) from, (lds_ptr_t) (uintptr_t) (cells + at), 16, 0, 0);
    }
    asm volatile("" ::: "memory");

    // This lane's granules of a piece: at[i] bytes on in row from[i] of the tile that is
    // being loaded. (Every lane loads, so that the loads in flight are known: a place that
    // holds none of a row's granules gets its last one again.)
    int32_t at[NL];
    const uint8_t * from[NL];
#pragma unroll
    for (int i = 0; i < NL; i++) {
        const int p = i * 64 + lane;
        at[i] = min(p - (p / GP) * GP, G - 1) * 16;
    }
    auto rows_from = [&](int tile) {
#pragma unroll
        for (int i = 0; i < NL; i++) {
            const int r = min((i * 64 + lane) / GP, 16 * S - 1);
            const call_row c = row_of(a, min(first_row + tile * 16 + (r & 15), end_row - 1));
            from[i] = (S == 1 ? pick(a.w, c.weight) : r >= 16 ? a.w[1] : a.w[0]) + (int64_t) c.row * row_bytes;
        }
    };
    // A granule holds bytes of its row: those before its first or behind its last that are
    // read with them are within the granule's own 16.
    struct place {
        int tile, piece;
    };
    auto load = [&](place p, int slot) {
        const uint32_t to = ring + slot * (NL * 1024);
        const int on = p.piece * (U * ST::UNIT);
        if (p.piece < pieces - 1) {
#pragma unroll
            for (int i = 0; i < NL; i++)
                __builtin_amdgcn_global_load_lds((global_ptr_t) (((uintptr_t) (from[i] + on) & ~(uintptr_t) 15) + at[i]), (lds_ptr_t) (uintptr_t) (to + i * 1024), 16, 0, 0);
        } else {  // behind a row's end, its last granule again
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const uintptr_t q = ((uintptr_t) (from[i] + on) & ~(uintptr_t) 15) + at[i], last = (uintptr_t) (from[i] + row_bytes - 1) & ~(uintptr_t) 15;
                __builtin_amdgcn_global_load_lds((global_ptr_t) (q < last ? q : last), (lds_ptr_t) (uintptr_t) (to + i * 1024), 16, 0, 0);
            }
        }
    };
    auto after = [&](place p) {
        p.piece++;
        if (p.piece == pieces) {
            p.piece = 0;
            p.tile++;
        }
        return p;
    };
    place now{u0 / pieces, 0};
    now.piece = u0 - now.tile * pieces;
    place then = now;
    // (a wave without that many pieces loads what follows, or the last)
    rows_from(min(then.tile, tiles - 1));
#pragma unroll
    for (int r = 0; r < RING; r++) {
        load(then, r);
        then = after(then);
        if (then.piece == 0) rows_from(min(then.tile, tiles - 1));
        asm volatile("" ::: "memory");
    }
    // x is there: this wave's loads of it, then (READY) everybody's
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(RING * NL) : "memory");
    if (threadIdx.x == 0) lds(zeros, u32x4{0, 0, 0, 0});
    if constexpr (!READY) {  // the cells that the wave has loaded, each over its own values, which its eight lanes have read
        for (uint32_t at = wave * 1024; at < cell_bytes; at += STREAM_WAVES * 1024) {
            const f32x4 v = lds<f32x4>(cells + at + lane * 16);
            const prepared r = prepare(make_float4(v.x, v.y, v.z, v.w));
            const int j = lane & 7;
            const uint32_t cell = cells + at + (lane >> 3) * RAW_CELL;
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
            for (int d = 0; d < 3; d++) lds(cell + (j >> 2) * 48 + d * 16 + (j & 3) * 4, r.digits[d]);
            if (j == 0) lds(cell + 96, f32x2{r.factor, r.sum});
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();  // (not __syncthreads, which waits for the weights too)
    asm volatile("" ::: "memory");

    float acc[M][S];
    auto clear = [&]() {
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int s = 0; s < S; s++) acc[m][s] = 0.0f;
    };
    uint32_t begins[S];  // where this lane's row begins in its first granule
    auto rows_of_tile = [&](int tile) {
        if constexpr (ALIGN < 16) {
            const call_row c = row_of(a, min(first_row + tile * 16 + col, end_row - 1));
#pragma unroll
            for (int s = 0; s < S; s++) begins[s] = (uint32_t) (uintptr_t) (S == 1 ? pick(a.w, c.weight) : a.w[s]) + (uint32_t) c.row * (uint32_t) row_bytes;
        }
    };
    const bool digit = (col >> 2) == group && (col & 3) < 3;
    const int ragged = a.chunks - (pieces - 1) * (STEPS * GROUPS) < STEPS * GROUPS ? pieces - 1 : pieces;  // the piece that is not whole
    // What a step takes from shared memory: requested a step ahead.
    struct operands {
        typename Q::raw w[S];
        i32x4 x[M][B][2];
        f32x2 f[M][B];  // the factor and the sum
    };
    auto compute = [&](int piece, uint32_t slot, auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        uint32_t unit[S];
#pragma unroll
        for (int s = 0; s < S; s++) unit[s] = slot + (s * 16 + col) * (GP * 16) + (ALIGN < 16 ? (begins[s] + (uint32_t) piece * (U * ST::UNIT)) & 15 : 0);
        const int step0 = piece * STEPS;
        auto request = [&](int i, operands & o) {
#pragma unroll
            for (int s = 0; s < S; s++)  // (past the row's end: any bytes, whose scales are then replaced)
                o.w[s] = ST::read(unit[s] + i / (ST::CHUNKS / GROUPS) * ST::UNIT, (i % (ST::CHUNKS / GROUPS)) * GROUPS + group);
            const bool in = !EDGE || (step0 + i) * GROUPS + group < a.chunks;
            const uint32_t cell = cells + (EDGE ? min((step0 + i) * GROUPS + group, a.chunks - 1) : (step0 + i) * GROUPS + group) * (B * M * CELL_AT);
            const uint32_t x_at = digit && in ? cell + (col & 3) * 16 : zeros;
            const uint32_t stride = digit && in ? CELL_AT : 0, part = digit && in ? 48 : 0;
#pragma unroll
            for (int m = 0; m < M; m++)
#pragma unroll
                for (int b = 0; b < B; b++) {
                    o.x[m][b][0] = lds<i32x4>(x_at + (b * M + m) * stride);
                    o.x[m][b][1] = lds<i32x4>(x_at + (b * M + m) * stride + part);
                    o.f[m][b] = lds<f32x2>(cell + (b * M + m) * CELL_AT + 96);
                }
        };
        operands o[2];
        request(0, o[0]);
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            if (i + 1 < STEPS) request(i + 1, o[(i + 1) & 1]);
            asm volatile("" ::: "memory");
            const operands & now = o[i & 1];
            const int chunk = (step0 + i) * GROUPS + group;
#pragma unroll
            for (int s = 0; s < S; s++) {
                uint32_t c[B][2][4];
                Q::codes(now.w[s], c);
                block_scales<B> sc = Q::scales(now.w[s], chunk);
#pragma unroll
                for (int b = 0; b < B; b++) {
                    if (EDGE && chunk >= a.chunks) sc.scale[b] = sc.offset[b] = 0.0f;
                    i32x4 d[M];
#pragma unroll
                    for (int m = 0; m < M; m++)
                        d[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.x[m][b][0], i32x4{(int) c[b][0][0], (int) c[b][0][1], (int) c[b][0][2], (int) c[b][0][3]}, i32x4{}, 0, 0, 0);
#pragma unroll
                    for (int m = 0; m < M; m++)
                        d[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(now.x[m][b][1], i32x4{(int) c[b][1][0], (int) c[b][1][1], (int) c[b][1][2], (int) c[b][1][3]}, d[m], 0, 0, 0);
#pragma unroll
                    for (int m = 0; m < M; m++) {
                        // (nibbles' sums |d0| <= 127 8 32 and |d1|, |d2| <= 128 8 32 fit in 32 bits together)
                        const float v = Q::NIBBLES ? (float) ((((d[m][0] << 8) + d[m][1]) << 8) + d[m][2]) : fmaf((float) d[m][0], 65536.0f, (float) ((d[m][1] << 8) + d[m][2]));
                        acc[m][s] = fmaf(v, sc.scale[b] * now.f[m][b].x, acc[m][s]);
                        if constexpr (Q::OFFSETS) acc[m][s] = fmaf(now.f[m][b].y, sc.offset[b], acc[m][s]);
                    }
                }
            }
        }
    };
    // a wave's sums of a tile; waves share a tile with their neighbours, so a tile's
    // place plus the wave's number is each result's own place
    auto leave = [&](int tile) {
        float * const to = red + (tile + wave) * (M * S * 16);
#pragma unroll
        for (int m = 0; m < M; m++)
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float v = over_groups(acc[m][s]);
                if (group == 0) to[(m * S + s) * 16 + col] = v;
            }
    };
    clear();
    rows_of_tile(now.tile);
    int slot = 0;
    for (int u = u0; u < u1; u++) {
        // the piece is there when no more than the loads after it are on their way (the
        // first RING are requested whether or not there are as many)
        if (u + RING <= u1 || u == u0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 1) * NL) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (now.piece == ragged) compute(now.piece, ring + slot * (NL * 1024), std::true_type{});
        else compute(now.piece, ring + slot * (NL * 1024), std::false_type{});
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before it is overwritten
        if (u + RING < u1) {
            load(then, slot);
            then = after(then);
            if (then.piece == 0) rows_from(min(then.tile, tiles - 1));
        }
        slot = slot + 1 == RING ? 0 : slot + 1;
        const place next = after(now);
        if (next.piece == 0 || u + 1 == u1) {
            leave(now.tile);
            clear();
            rows_of_tile(next.tile);
        }
        now = next;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (nothing is on its way to a wave that has ended)
    __syncthreads();
    for (int i = threadIdx.x; i < tiles * M * 16; i += STREAM_WAVES * 64) {
        const int c = i & 15, m = (i >> 4) % M, k = (i >> 4) / M, r = first_row + k * 16 + c;
        if (r >= end_row) continue;
        float v[S];
#pragma unroll
        for (int s = 0; s < S; s++) v[s] = 0.0f;
#pragma unroll
        for (int w = 0; w < STREAM_WAVES; w++) {
            const bool has = max(waves.start(w), k * pieces) < min(waves.start(w + 1), (k + 1) * pieces);
#pragma unroll
            for (int s = 0; s < S; s++) {
                const float one = red[(k + w) * (M * S * 16) + (m * S + s) * 16 + c];
                v[s] += has ? one : 0.0f;
            }
        }
        const call_row to = row_of(a, r);
        store_row<S>(a, to.weight, to.row, m, v);
    }
}

// ---- the host's plan ----------------------------------------------------------------

struct matvec_plan {
    int ring;             // of stream_kernel; 0: matvec_kernel
    int wk, wr, height, workgroups, seg_steps, segs, pieces;
    bool copy;            // of stream_kernel: x is prepared by a kernel of its own
    size_t lds, bytes;
};

// Streams' sizes by type, as the kernels have them.
struct stream_sizes {
    int pieces, loads;
};
template <int S> stream_sizes sizes_of(int type, int chunks) {
#define ZEST_SIZES(T) \
    case T: return {(chunks + stream<T>::CHUNKS * UNITS<S> - 1) / (stream<T>::CHUNKS * UNITS<S>), LOADS<T, S>}
    switch (type) {
        ZEST_SIZES(ZEST_TYPE_Q4_0);
        ZEST_SIZES(ZEST_TYPE_Q4_1);
        ZEST_SIZES(ZEST_TYPE_Q8_0);
        ZEST_SIZES(ZEST_TYPE_Q4_K);
        ZEST_SIZES(ZEST_TYPE_IQ4_NL);
        default: ZEST_SIZES(ZEST_TYPE_IQ4_XS);
    }
#undef ZEST_SIZES
}

// Tiles' sizes by type: a block's cell, a wave's own shared memory.
struct tile_sizes {
    int cell, wave;
};
tile_sizes tile_sizes_of(int type, int height) {
#define ZEST_SIZES(T) \
    case T: return {TILE_CELL<T>, height == 2 ? WAVE_BYTES<T, 2> : WAVE_BYTES<T, 1>}
    switch (type) {
        ZEST_SIZES(ZEST_TYPE_Q4_0);
        ZEST_SIZES(ZEST_TYPE_Q4_1);
        ZEST_SIZES(ZEST_TYPE_Q8_0);
        ZEST_SIZES(ZEST_TYPE_Q4_K);
        ZEST_SIZES(ZEST_TYPE_IQ4_NL);
        default: ZEST_SIZES(ZEST_TYPE_IQ4_XS);
    }
#undef ZEST_SIZES
}

constexpr int CUS = 256;
constexpr int STREAM_ROWS = 512;  // of a workgroup at most

matvec_plan plan_of(int type, int64_t M, int64_t K, int n, const int64_t * N, bool glu) {
    matvec_plan p{};
    const int B = type == ZEST_TYPE_Q4_K ? 2 : 1, chunks = (int) (K / 32 / B), steps = (chunks + GROUPS - 1) / GROUPS, S = glu ? 2 : 1;
    if (M <= 4) {
        const stream_sizes z = glu ? sizes_of<2>(type, chunks) : sizes_of<1>(type, chunks);
        int64_t rows = 0;
        for (int i = 0; i < (glu ? 1 : n); i++) rows += N[i];
        p.pieces = z.pieces;
        p.workgroups = (int) std::max<int64_t>(std::min<int64_t>(rows, CUS), (rows + STREAM_ROWS - 1) / STREAM_ROWS);
        const int64_t wg_tiles = ((rows + p.workgroups - 1) / p.workgroups + 15) / 16;
        const auto lds_of = [&](int ring, int cell) {
            return (size_t) STREAM_WAVES * ring * z.loads * 1024 + (((size_t) B * chunks * M * cell + 1023) & ~(size_t) 1023) + 16 +
                   (size_t) (wg_tiles + STREAM_WAVES) * M * S * 16 * 4;
        };
        for (p.ring = 3; p.ring >= 2; p.ring--)
            for (const int cell : {RAW_CELL, CELL}) {
                p.lds = lds_of(p.ring, cell);
                p.copy = cell == CELL;
                p.bytes = p.copy ? (size_t) B * chunks * M * CELL : 0;
                if (p.lds <= LDS_MOST && (p.ring == 2 || !p.copy)) return p;
            }
        p.ring = 0;
    }
    // 32 rows a tile where there are enough of them: x is read from shared memory half as often
    int64_t wide = 0, narrow = 0;
    for (int i = 0; i < (glu ? 1 : n); i++) wide += (N[i] + 31) / 32, narrow += (N[i] + 15) / 16;
    p.height = glu || wide > 4 * CUS ? 2 : 1;
    const int64_t tiles = glu || p.height == 1 ? narrow : wide;
    p.wr = tiles <= 2 * CUS ? 1 : tiles <= 8 * CUS ? 2 : 4;
    const int most = p.wr == 1 && tiles > CUS ? 8 : 16 / p.wr;
    p.wk = 1;
    for (int w = 1; w <= most; w++)
        if ((steps + w - 1) / w < (steps + p.wk - 1) / p.wk) p.wk = w;
    const tile_sizes z = tile_sizes_of(type, p.height);
    const size_t cell = z.cell, own = (size_t) p.wk * p.wr * z.wave;
    p.seg_steps = (int) std::min<size_t>(steps, (LDS_MOST - own) / ((size_t) GROUPS * B * cell));
    p.segs = (steps + p.seg_steps - 1) / p.seg_steps;
    p.lds = (size_t) std::min(p.seg_steps * GROUPS, chunks) * B * cell + own;
    p.workgroups = (int) std::min<int64_t>((tiles + p.wr - 1) / p.wr, 2 * CUS);
    if (p.lds > LDS_MOST / 2 || p.wk * p.wr > 8) p.workgroups = std::min(p.workgroups, CUS);
    p.bytes = (size_t) chunks * B * cell;
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

template <int BYTES> void launch_prepare(const matvec_args & a, hipStream_t s) {
    hipLaunchKernelGGL(prepare_kernel<BYTES>, dim3((unsigned) std::min<int64_t>(((int64_t) a.blocks * a.M * 8 + 255) / 256, 1024)), dim3(256), 0, s, a);
}

template <int TYPE, int H, int S> int launch(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (const int st = allow_lds<&matvec_kernel<TYPE, H, S>>(me)) return st;
    launch_prepare<TILE_CELL<TYPE>>(a, s);
    hipLaunchKernelGGL((matvec_kernel<TYPE, H, S>), dim3((unsigned) p.workgroups), dim3((unsigned) (p.wk * p.wr * 64)), p.lds, s, a);
    return zest::check_launch(me);
}

template <int TYPE, int M, int S, int RING, bool READY> int launch_stream(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (const int st = allow_lds<&stream_kernel<TYPE, M, S, RING, READY>>(me)) return st;
    if (READY) launch_prepare<CELL>(a, s);
    hipLaunchKernelGGL((stream_kernel<TYPE, M, S, RING, READY>), dim3((unsigned) p.workgroups), dim3(STREAM_WAVES * 64), p.lds, s, a);
    return zest::check_launch(me);
}

template <int TYPE, int M, int S> int launch_stream(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (p.copy) return launch_stream<TYPE, M, S, 2, true>(a, p, s, me);
    return p.ring == 3 ? launch_stream<TYPE, M, S, 3, false>(a, p, s, me) : launch_stream<TYPE, M, S, 2, false>(a, p, s, me);
}

template <int TYPE, int S> int launch(const matvec_args & a, const matvec_plan & p, hipStream_t s, const char * me) {
    if (p.ring) {
        if (a.M > 2) return a.M > 3 ? launch_stream<TYPE, 4, S>(a, p, s, me) : launch_stream<TYPE, 3, S>(a, p, s, me);
        return a.M > 1 ? launch_stream<TYPE, 2, S>(a, p, s, me) : launch_stream<TYPE, 1, S>(a, p, s, me);
    }
    if constexpr (S == 1)
        if (p.height == 1) return launch<TYPE, 1, 1>(a, p, s, me);
    return launch<TYPE, 2, S>(a, p, s, me);
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
    a.blocks = (int32_t) (K / 32);
    a.chunks = a.blocks / (type == ZEST_TYPE_Q4_K ? 2 : 1);
    a.n = outs;
    a.glu = glu;
    int64_t rows = 0;
    for (int i = 0; i < n; i++) {
        ZEST_REQUIRE(w[i] && aligned(w[i], row_align(type)), "%s: weight %d: rows %d-byte aligned wanted", me, i, row_align(type));
        ZEST_REQUIRE(N[i] > 0 && N[i] <= (1 << 26), "%s: weight %d: N=%lld", me, i, (long long) N[i]);
        a.w[i] = (const uint8_t *) w[i];
        a.N[i] = (int32_t) N[i];
        if (i < outs) rows += N[i];
        a.rows[i] = (int32_t) rows;
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
    const matvec_plan p = plan_of(type, M, K, n, N, glu >= 0);
    ZEST_REQUIRE(!p.bytes || (workspace && aligned(workspace, 16) && workspace_bytes >= p.bytes), "%s: workspace of %zu bytes, 16-byte aligned, wanted", me, p.bytes);
    const int tile_rows = glu < 0 && p.height == 2 ? 32 : 16;
    for (int i = 0; i < outs; i++) a.tiles[i] = a.all_tiles += (int32_t) ((N[i] + tile_rows - 1) / tile_rows);
    a.wk = p.wk, a.wr = p.wr, a.seg_steps = p.seg_steps, a.segs = p.segs;
    a.cells = (uint8_t *) workspace;
    a.pieces = p.pieces, a.each = (int32_t) (rows / p.workgroups), a.more = (int32_t) (rows % p.workgroups);
    return launch(type, a, p, zest::as_stream(stream), me);
}

} // namespace

extern "C" {

size_t zest_matvec_workspace(int type, int64_t M, int64_t K, int n, const int64_t * N) {
    if (!supported(type) || M <= 0 || M > MAX_M || K <= 0 || K > (1 << 20) || !zest_raw_row_bytes(type, K) || n < 1 || n > MAX_N || !N) return 0;
    for (int i = 0; i < n; i++)
        if (N[i] <= 0 || N[i] > (1 << 26)) return 0;
    const size_t bytes = plan_of(type, M, K, n, N, false).bytes;
    return n == 2 && N[0] == N[1] ? std::max(bytes, plan_of(type, M, K, n, N, true).bytes) : bytes;
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

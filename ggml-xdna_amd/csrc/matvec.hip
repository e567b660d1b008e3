// Products of a few rows with GGUF weights as they are (include/zest/decode.h):
// y[m][n] = sum_k x[m][k] W[n][k], HBM bound by the weights' bytes.
//
// A chunk is 32 of a weight row's values, of which 16 bytes of codes hold two
// halves of 16: the low and the high nibbles (Q8_0: 32 bytes, its first and last
// 16). Every half is code * scale + offset, codes signed bytes.
#include <algorithm>

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

struct matvec_args {
    const float * x;
    int64_t ldx, row_bytes;
    int32_t M, chunks, n, glu;   // chunks of a row; glu: the kind, -1: none
    const uint8_t * w[MAX_N];
    const float * res[MAX_N];
    float * y[MAX_N];
    int64_t ldy[MAX_N], ldr[MAX_N];
    int32_t N[MAX_N];
    int32_t rows;                // output rows in all (of a GLU: of one weight)
};

// A wave an output row (a pair of them for a GLU), a lane every 64th chunk.
template <int TYPE> __device__ inline void dot_row(const matvec_args & a, const uint8_t * row, float acc[MAX_M]) {
    typedef quant<TYPE> Q;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 0; m < MAX_M; m++) acc[m] = 0.0f;
    for (int c = lane; c < a.chunks; c += 64) {
        const typename Q::raw r = Q::load(row, c);
        uint32_t q[2][4];
        Q::codes(r, q);
        const half_scales s = Q::scales(r, c);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float * x = a.x + half_column<TYPE>(c, h);
#pragma unroll
            for (int m = 0; m < MAX_M; m++) {
                if (m >= a.M) continue;
                float dot = 0.0f, sum = 0.0f, odd = 0.0f;  // odd: NaN where a value of x is not finite
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float4 v = *reinterpret_cast<const float4 *>(x + m * a.ldx + 4 * i);
                    const float e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        dot = fmaf(e[j], (float) (int8_t) (q[h][i] >> 8 * j), dot);
                        sum += e[j];
                        odd = fmaf(e[j], 0.0f, odd);
                    }
                }
                acc[m] = fmaf(dot, s.scale[h], fmaf(sum, s.offset[h], acc[m])) + odd;
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MAX_M; m++)
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) acc[m] += __shfl_xor(acc[m], off);
}

template <int TYPE> __global__ __launch_bounds__(256) void matvec_kernel(matvec_args a) {
    int64_t row = (int64_t) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows) return;
    int i = 0;
    if (a.glu < 0)
        while (row >= a.N[i]) row -= a.N[i++];
    float acc[MAX_M], up[MAX_M];
    dot_row<TYPE>(a, a.w[i] + row * a.row_bytes, acc);
    if (a.glu >= 0) dot_row<TYPE>(a, a.w[1] + row * a.row_bytes, up);
    if ((threadIdx.x & 63) != 0) return;
    for (int m = 0; m < MAX_M; m++) {
        if (m >= a.M) continue;
        float v = a.glu >= 0 ? zest::glu(a.glu, acc[m], up[m]) : acc[m];
        if (a.res[i]) v += a.res[i][m * a.ldr[i] + row];
        a.y[i][m * a.ldy[i] + row] = v;
    }
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

int launch(int type, const matvec_args & a, hipStream_t s, const char * me) {
    const dim3 grid((unsigned) ((a.rows + 3) / 4)), block(256);
    switch (type) {
        case ZEST_TYPE_Q4_0: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_Q4_0>, grid, block, 0, s, a); break;
        case ZEST_TYPE_Q4_1: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_Q4_1>, grid, block, 0, s, a); break;
        case ZEST_TYPE_Q8_0: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_Q8_0>, grid, block, 0, s, a); break;
        case ZEST_TYPE_Q4_K: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_Q4_K>, grid, block, 0, s, a); break;
        case ZEST_TYPE_IQ4_NL: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_IQ4_NL>, grid, block, 0, s, a); break;
        default: hipLaunchKernelGGL(matvec_kernel<ZEST_TYPE_IQ4_XS>, grid, block, 0, s, a); break;
    }
    return zest::check_launch(me);
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
    a.n = n;
    a.glu = glu;
    int64_t rows = 0;
    for (int i = 0; i < n; i++) {
        ZEST_REQUIRE(w[i] && aligned(w[i], row_align(type)), "%s: weight %d: rows %d-byte aligned wanted", me, i, row_align(type));
        ZEST_REQUIRE(N[i] > 0 && N[i] <= (1 << 26), "%s: weight %d: N=%lld", me, i, (long long) N[i]);
        a.w[i] = (const uint8_t *) w[i];
        a.N[i] = (int32_t) N[i];
        if (i < outs) rows += N[i];
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
    ZEST_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= zest_matvec_workspace(type, M, K, n, N), "%s: workspace of %zu bytes, 16-byte aligned, wanted", me,
                 zest_matvec_workspace(type, M, K, n, N));
    a.rows = (int32_t) rows;
    return launch(type, a, zest::as_stream(stream), me);
}

} // namespace

extern "C" {

size_t zest_matvec_workspace(int type, int64_t M, int64_t K, int n, const int64_t * N) {
    if (!supported(type) || M <= 0 || M > MAX_M || K <= 0 || K > (1 << 20) || n < 1 || n > MAX_N || !N) return 0;
    return 16;
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

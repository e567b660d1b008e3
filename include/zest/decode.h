/*
 * zest/decode.h — the C ABI of a decoding step's other kernels (attention over
 * the paged cache is in zest/kv.h): products of a few rows with GGUF weights as
 * they are, and the choice of the next token. In the manner of zest_hip.h:
 * plain pointers, sizes and status codes; every call checks its arguments on the
 * host, enqueues work on `stream` of the current device and returns; nothing is
 * allocated and no call waits for the GPU, so all of them may be captured in a
 * HIP graph. The reference leaves a decoding step to other backends (its gate
 * claims matmuls of 1024 rows and more), so these have no counterpart in it.
 *
 * Workspaces are the caller's, 16-byte aligned, of the size that a host call
 * gives by sizes alone (0: none is wanted, and NULL will do). They hold nothing
 * between calls; calls that may overlap (on two streams, or as replays of two
 * graphs) need one each.
 */
#ifndef ZEST_DECODE_H
#define ZEST_DECODE_H

#include "../zest_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* y[i][M][N[i]] = x . W_i^T (+ res[i]) for up to ZEST_MATVEC_MAX_GROUP weights on
 * one x in one launch: x fp32 rows of K values, W_i GGUF rows of `type` (Q4_0,
 * Q4_1, Q4_K, IQ4_NL, IQ4_XS or Q8_0; N[i] rows of zest_raw_row_bytes(type, K)
 * bytes each) as a model file holds them, y and res fp32 rows. The values the
 * weights stand for are used exactly, x to 2^-22 of the largest magnitude in its
 * 32 (groups of consecutive values), sums are in fp32, in an order that a call's
 * sizes fix. A row of x that holds a NaN or an infinity gives NaN in all of its y
 * row.
 *
 * M 1 .. ZEST_MATVEC_MAX_ROWS (more rows: zest_gemm), K a multiple of the type's
 * block (32, or 256 for Q4_K and IQ4_XS) up to 2^20, N[i] up to 2^26. x rows
 * 16-byte aligned (ldx floats apart); W rows aligned as for zest_convert_weight;
 * y and res 4-byte aligned. res may be NULL, or hold NULLs; res[i] may be y[i]
 * itself (equal strides). A y must not overlap x, a weight, another y, or a res
 * otherwise (columns of one wider buffer, equal strides, do not). */
#define ZEST_MATVEC_MAX_ROWS 16
#define ZEST_MATVEC_MAX_GROUP 4
ZEST_API size_t zest_matvec_workspace(int type, int64_t M, int64_t K, int n, const int64_t *N);
ZEST_API int zest_matvec(int type, const float *x, int64_t M, int64_t K, int64_t ldx, int n, const void *const *w,
                         const int64_t *N, const float *const *res, const int64_t *ldr, float *const *y,
                         const int64_t *ldy, void *workspace, size_t workspace_bytes, void *stream);

/* y[M][F] = glu(x . gate^T, x . up^T) of `kind` (zest_glu's arithmetic, over the
 * sums zest_matvec gives): two weights of F rows in one launch. The workspace is
 * zest_matvec_workspace's for n = 2, N = {F, F}. */
ZEST_API int zest_matvec_glu(int kind, int type, const float *x, int64_t M, int64_t K, int64_t ldx, const void *gate,
                             const void *up, int64_t F, float *y, int64_t ldy, void *workspace, size_t workspace_bytes,
                             void *stream);

/* The next token of each row of logits[rows][vocab] (F32, F16 or BF16, ld values
 * apart), from the random number u[row] in [0, 1):
 *   1. weights w_i = exp((x_i - max x) / temperature), the largest exactly 1;
 *   2. top_k: the k largest logits stay (ties: the lower index first);
 *   3. top_p: of those, in that order, the shortest run that holds at least
 *      top_p of their weight stays;
 *   4. min_p: of those, weights of at least min_p stay;
 *   5. token[row] is the first index, in index order, whose running sum of what
 *      stays exceeds u times all of it, and prob[row] (NULL: not wanted) its
 *      share of that.
 * Weights are computed in 64 bits and summed as 64-bit integers of 2^-45 of the
 * largest, so a result does not depend on the order of a sum.
 *
 * temperature, top_k, top_p, min_p (device, one a row; NULL: 1 and off):
 * a temperature that is not above 0 takes the largest logit (the lowest index
 * of several; probability 1); top_k <= 0, top_p >= 1 and min_p <= 0 are off, as is a NaN;
 * top_p <= 0 leaves the largest, min_p > 1 counts as 1. u below 0 (or NaN) counts
 * as 0, from 1 on the last token that stays is taken. A logit of -infinity or NaN
 * is never taken; logits of +infinity share all the weight. A row without any
 * logit above -infinity gives token -1 and probability 0.
 *
 * vocab 1 .. 2^18, rows 1 .. 65536; logits aligned to their type. */
#define ZEST_SAMPLE_MAX_VOCAB (1 << 18)
ZEST_API size_t zest_sample_workspace(int64_t rows, int64_t vocab);
ZEST_API int zest_sample(const void *logits, int type, int64_t rows, int64_t vocab, int64_t ld, const float *u,
                         const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                         int32_t *token, float *prob, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif

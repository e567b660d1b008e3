/*
 * zest/kv.h — the paged KV cache: the C ABI of the kernels that append a
 * chunk's keys and values to it, attend over it, and keep its pages. In the
 * manner of zest_hip.h: plain pointers, sizes and status codes; every call
 * checks its arguments on the host, enqueues work on `stream` of the current
 * device and returns; nothing is allocated, and no call waits for the GPU, so
 * all of them may be captured in a HIP graph. It has no counterpart in the
 * reference, whose offload stops at the matmuls on either side of attention.
 *
 * The cache. A layer's pool is `pages` pages of page_tokens tokens, all k/v
 * heads of them. A page is, head after head, K as [head_dim/8][page_tokens][8]
 * and then V as [page_tokens/16][2][head_dim][8]: the 8 values of a K piece are
 * one token's, the 8 of a V piece are one column's, for tokens 4h..4h+3 and
 * 8+4h..8+4h+3 of the 16 (h the second index). Both are the order in which
 * v_mfma_f32_32x32x16 takes them, so a fragment is 16 contiguous bytes a lane.
 * A slot is a sequence: its row of `tables` names its pages in order, its entry
 * of `lens` counts its tokens, and refs[page] counts the rows that name a page.
 * Layers share tables, lens and refs; their pools lie layer_stride bytes apart.
 *
 * Device-side contents (tables, lens, starts, slots and lists) are checked on
 * the device: what they name outside the pool, the tables, the rows or the
 * bounds given is not read or written, and `*bad` (a device word, NULL: not
 * reported) is OR-ed with 1.
 */
#ifndef ZEST_KV_H
#define ZEST_KV_H

#include "../zest_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
    void *pool;          /* one layer's pages, 16-byte aligned */
    int64_t pages;       /* 1 .. 2^24 */
    int32_t type;        /* ZEST_TYPE_F16 or ZEST_TYPE_BF16 */
    int32_t kv_heads;    /* 1 .. 1024 */
    int32_t head_dim;    /* 64, 96, 128, 192 or 256 */
    int32_t page_tokens; /* 16, 32, 64, 128 or 256 */
} zest_kv_cache;

/* The sequences of one call. Sequence b is slot slots[b] (b itself where slots
 * is NULL); its new tokens are rows starts[b] .. starts[b+1]-1 of q, k, v and
 * the output, and the last of its lens[slot] tokens: row i of n is token
 * lens[slot] - n + i. Rows outside every sequence's are neither read nor
 * written. max_new and max_len bound n and lens from above: a sequence beyond
 * them is left out and reported. Starts do not decrease: where they do, that is
 * reported, and other sequences may be left out with the one it is seen at. */
typedef struct {
    const int32_t *tables; /* [table_rows][table_cols], device */
    const int32_t *lens;   /* [table_rows], device */
    const int32_t *starts; /* [seqs + 1], device */
    const int32_t *slots;  /* [seqs], device, or NULL */
    int64_t rows;          /* rows of q, k, v and the output, 1 .. 2^27 */
    int32_t seqs;          /* 1 .. 4096 */
    int32_t table_rows, table_cols;
    int32_t max_new;       /* 1 .. rows */
    int32_t max_len;       /* 0 .. 2^30 */
} zest_kv_batch;

/* Rotary positions: pair p of the first n_dims of a head turns by position *
 * freqs[p], the product and its reduction in 64 bits (32 lose the angle of far
 * positions), and is multiplied by magnitude. mode 0: pair p is dims 2p and
 * 2p+1; mode 2 (NeoX): p and n_dims/2 + p. */
typedef struct {
    const double *freqs; /* [n_dims/2], device */
    int32_t n_dims;      /* even, <= head_dim */
    int32_t mode;
    float magnitude;
} zest_kv_rope;

ZEST_API size_t zest_kv_page_bytes(const zest_kv_cache *cache);

/* The frequencies zest_rope's parameters stand for, as a table for
 * zest_kv_rope (host arithmetic, out[n_dims/2] on the host): freq_base^(-2p /
 * n_dims) / ff[p], interpolated by freq_scale and, with ext_factor, mixed with
 * the extrapolated one as YaRN does between the correction dims. Returns the
 * magnitude (attn_factor, and YaRN's 1 + 0.1 ln(1 / freq_scale)) in
 * *magnitude. */
ZEST_API int zest_kv_rope_freqs(int32_t n_dims, double freq_base, double freq_scale, double ext_factor,
                                double attn_factor, double corr0, double corr1, const float *ff, double *out,
                                float *magnitude);

/* The new tokens' keys and values into their pages: k (turned by `rope`, NULL:
 * as it is) and v, rows of kv_heads * head_dim values of in_type (F32, F16 or
 * BF16), ldk and ldv values apart, rounded once to the cache's type. With q,
 * also q's rows of q_heads * head_dim turned by the same angles into q_out (of
 * q_out_type; q_out may be q itself where types and strides agree, and must not
 * overlap q otherwise, nor k, v or the pool: columns of one wider buffer, equal
 * strides, do not). The angle's position is the token's place in its sequence, or pos[row] (device, NULL: the
 * place). Row starts of q, k, v and q_out 16-byte aligned. A token whose place
 * is negative (lens below the new tokens) or whose page is not in the pool is
 * not stored, and reported; its q row is still turned. Two sequences of a call
 * must not name the same slot. */
ZEST_API int zest_kv_append(const zest_kv_cache *cache, const zest_kv_batch *batch, const zest_kv_rope *rope,
                            const int32_t *pos, int in_type, const void *k, int64_t ldk, const void *v, int64_t ldv,
                            const void *q, int64_t ldq, int32_t q_heads, void *q_out, int64_t ldq_out, int q_out_type,
                            uint32_t *bad, void *stream);

/* Attention of the new tokens over their sequences' tokens: for row i and query
 * head j (k/v head j / (q_heads / kv_heads)),
 *     out = sum_t softmax_t(s_t) v_t,  s_t = scale q.k_t,
 *     with softcap > 0: s_t = softcap tanh(scale q.k_t / softcap) (a softcap whose
 *     quotient scale / softcap passes 10^38 is refused),
 * over the tokens t < len that the row sees: with `causal` t <= its place, with
 * window > 0 also t > its place - window. Without `causal` every row sees the
 * whole sequence (an encoder's states: lens need not hold the rows). A row that
 * sees no token, or only scores of -infinity, is zero. Tokens that a row does
 * not see, and places behind len, do not reach it whatever they hold (NaN and
 * infinities too); pages of which no row sees a token may be gone from the table.
 * A page outside the pool counts as unseen and is reported.
 *
 * q_type and out_type: F32, F16 or BF16; q is rounded to the cache's type (the
 * matrix cores' operand), products and softmax statistics are in 32 bits, the
 * weights are rounded to the cache's type before they meet V. q_heads % kv_heads
 * == 0; row starts of q and out 16-byte aligned; out must not overlap q or the
 * pool (columns of one wider buffer, equal strides, do not).
 *
 * workspace: zest_kv_attn_workspace's bytes for the same cache, batch and
 * q_heads (by sizes and bounds alone), 16-byte aligned. It holds nothing between
 * calls; calls that may overlap need one each. A sum over keys that is split
 * among workgroups is joined in a fixed order, so a call's result does not vary
 * from run to run. */
ZEST_API size_t zest_kv_attn_workspace(const zest_kv_cache *cache, const zest_kv_batch *batch, int32_t q_heads);
ZEST_API int zest_kv_attn(const zest_kv_cache *cache, const zest_kv_batch *batch, const void *q, int q_type,
                          int64_t ldq, int32_t q_heads, float scale, int causal, int32_t window, float softcap,
                          void *out, int out_type, int64_t ldo, void *workspace, size_t workspace_bytes, uint32_t *bad,
                          void *stream);

/* Sequences that share what they say first: group g is the sequences
 * starts[g] .. starts[g+1]-1 of a batch (device; they do not decrease; a sequence
 * outside all groups shares nothing). What a group shares is found on the device:
 * the leading whole pages that the tables of all its members name alike, as far as
 * all its rows see all of them, and max_shared tokens at most. So a group is only
 * ever a hint, and forks of one prompt (zest_kv_assign) one after the other in a
 * batch are such a group. Unless `always` is set, groups that by the sizes and bounds
 * alone save too little to pay for the search and the join are passed over. */
typedef struct {
    const int32_t *starts; /* [groups + 1], device */
    int32_t groups;        /* 1 .. 2048 */
    int32_t max_shared;    /* 0 .. 2^30 */
    int32_t always;        /* 0 or 1 */
} zest_kv_groups;

/* zest_kv_attn where the batch's sequences come in groups: the same result but for
 * the order in which its sums are rounded, what a group shares being read once for
 * all its rows and joined with what each sequence holds of its own. Arguments and
 * limits as zest_kv_attn's; groups' starts outside 0 .. seqs, or going back, are
 * reported, and no group shares anything then. table_rows * table_cols < 2^31. The
 * workspace is zest_kv_attn_shared_workspace's. */
ZEST_API size_t zest_kv_attn_shared_workspace(const zest_kv_cache *cache, const zest_kv_batch *batch,
                                              const zest_kv_groups *groups, int32_t q_heads);
ZEST_API int zest_kv_attn_shared(const zest_kv_cache *cache, const zest_kv_batch *batch, const zest_kv_groups *groups,
                                 const void *q, int q_type, int64_t ldq, int32_t q_heads, float scale, int causal,
                                 int32_t window, float softcap, void *out, int out_type, int64_t ldo, void *workspace,
                                 size_t workspace_bytes, uint32_t *bad, void *stream);

/* Scratch bytes of zest_kv_assign (n entries) and zest_kv_compact (n = 0). */
ZEST_API size_t zest_kv_scratch_bytes(int64_t pages, int32_t n);

/* A scheduling step: for every entry i, slot dst[i] becomes what slot src[i] was
 * before the call (-1: empty; dst[i] itself: what it is), grown by grow[i]
 * tokens. So (free, -1, n) admits a sequence, (child, parent, n) forks one,
 * (slot, slot, n) grows it and (slot, -1, 0) frees it. The pages of a row that
 * is replaced are released first (refs - 1, free at 0); a fork shares its
 * parent's full pages (refs + 1) and gets a copy of its open one, whole, in
 * every layer; further pages are the lowest-numbered free ones, in the order of
 * the entries. Entries of a row past its pages become -1. An entry of -1 among
 * its pages is one that a window has left and the program has given back: a
 * release passes it over and a fork takes it over. Reported are the open page
 * of a fork that is missing, and other numbers outside the pool.
 *
 * An entry is left undone and reported when it names a slot outside the tables
 * (src -1 apart), grows by a negative number or past table_cols pages, when dst
 * is listed twice (then neither is done), or when src is the dst of another
 * entry that replaces it. Where the free pages run out, the entries from the
 * first that does not fit on get none: a grown slot stays as it was, any other
 * is left empty, reported; entries that need no page are done. table_rows <=
 * 65536, n <= 65536. */
ZEST_API int zest_kv_assign(const zest_kv_cache *cache, int32_t layers, int64_t layer_stride, int32_t *refs,
                            int32_t *tables, int32_t *lens, int32_t table_rows, int32_t table_cols, const int32_t *dst,
                            const int32_t *src, const int32_t *grow, int32_t n, void *scratch, size_t scratch_bytes,
                            uint32_t *bad, void *stream);

/* Moves the live pages (refs > 0) to the front of the pool: with n of them,
 * the k-th live page at or past n goes to the k-th free page below n, in every
 * layer; refs and every table entry follow; *live (device) = n. The pages past
 * n are then free and hold what they held. refs_out and tables_out may be refs
 * and tables (in place) or buffers of their own, for a program that switches to
 * the new tables later: until then the old ones stay valid only for the pages
 * that did not move into them. An entry that names a page without references,
 * or outside the pool (-1 apart), becomes -1 and is reported. */
ZEST_API int zest_kv_compact(const zest_kv_cache *cache, int32_t layers, int64_t layer_stride, const int32_t *refs,
                             const int32_t *tables, int32_t table_rows, int32_t table_cols, int32_t *refs_out,
                             int32_t *tables_out, int32_t *live, void *scratch, size_t scratch_bytes, uint32_t *bad,
                             void *stream);

#ifdef __cplusplus
}
#endif
#endif

/*
 * pam_hip_attention.h -- entry points of libpam_hip.so for attention in one piece, its gradients, and the paged cache that a model
 * reads while decoding.  The reference composes attention from its products and softmax.  Conventions as in pam_hip.h; results share
 * no memory with each other or with what is read, unless it is said that they may.  Pointers to prefix, documents, slopes, pages, lengths
 * and counts are device pointers.
 */
#ifndef PAM_HIP_ATTENTION_H
#define PAM_HIP_ATTENTION_H

#include <stddef.h>

#include "pam_hip_block.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Values of every token's heads, [batch][tokens][heads][dim]: a head's values lie side by side, the other strides are free. */
typedef struct { const float *p; long sb, st, sh; } pam_hip_tokens;

/* What query i does with key j (positions: the queries are the last `tokens` of `keys` tokens):
 *   a = sum over d of (q_d (*) scale) (*) k_d
 *   cap > 0:  a = cap (*) tanh(a (/) cap) with tanh u = (1 - w) (/) (1 + w), w = 2^-(u (*) 2 log2 e), odd in u
 *   slopes:   a = a - slopes[head] (*) |i - j|
 *   e_ij = 2^(a (*) log2 e),   l_i = sum of e_ij,   y_id = (sum of e_ij (*) v_jd) (/) l_i
 * over the keys that it sees: j <= i if causal; |i - j| < window if window > 0; those and all j < prefix[batch entry] if prefix; of those,
 * if documents ([batch][keys]), the ones of its own document, which is not negative.  A query that sees no key has the result zero, and no
 * gradients.  Keys' and values' heads are shared by heads / kv_heads queries' heads in a row.
 * Weights below 2^-62 of the largest that came before them are none.  A score that is not a finite number, or is 2^127 or more, makes its query's
 * results NaN.  offset multiplies every PAM product and quotient, and lies in (0.75, 1.5); scale lies in (2^-40, 2^40), cap is 0 or in
 * (2^-20, 2^20).  dim is a multiple of four, up to 256, of which the first `values` values of every head
 * count; the others (at most three) have to be 1 in keys and values and may be anything elsewhere. */
typedef struct {
    long batch, tokens, keys, heads, kv_heads, dim, values;
    float scale, cap, offset;
    int causal;
    long window;
    const long long *prefix, *documents;
    const float *slopes;
} pam_hip_attention_shape;

/* y is contiguous.  stats, if not NULL, receives two floats for every query's head, [batch][tokens][heads][2]: a backward pass reads them. */
size_t pam_hip_attention_workspace_bytes(const pam_hip_attention_shape *shape);
int pam_hip_attention_fwd(const pam_hip_attention_shape *shape, const pam_hip_tokens *q, const pam_hip_tokens *k, const pam_hip_tokens *v,
                          float *y, float *stats, void *workspace, size_t workspace_bytes, void *stream);

/* Gradients for q, k and v (contiguous; dq, or dk and dv, may be NULL) from that of y: the chain of the primitives' gradients, with the
 * sums of heads that share a key.  y (contiguous) and stats are the forward pass's.  The approx flags are those of pam_hip_act_bwd.  Of approximate gradients a
 * pair's (that for a) is none below 2^-116 of the largest dy (*) (1 (/) l) of its query or, for dk and dv, of the queries that are worked on together. */
size_t pam_hip_attention_bwd_workspace_bytes(const pam_hip_attention_shape *shape, int want_q, int want_kv);
int pam_hip_attention_bwd(const pam_hip_attention_shape *shape, const pam_hip_tokens *q, const pam_hip_tokens *k, const pam_hip_tokens *v,
                          const float *y, const float *stats, const pam_hip_tokens *dy, float *dq, float *dk, float *dv,
                          int approx_a, int approx_b, int approx_exp, void *workspace, size_t workspace_bytes, void *stream);

/* A cache in pages: keys and values of [pages][page][kv_heads][dim], a head's values side by side, the other strides (the same for both) free.
 * pages ([batch][per_sequence], contiguous): the page of a sequence's places 0 ... page - 1, then of the next ones.  lengths ([batch]): the tokens of
 * every sequence that are in the cache already; token t of a call is at place lengths + t.  counts ([batch]) or NULL: how many of a call's tokens a
 * sequence has; the others are padding.  dim: up to 256. */
typedef struct {
    long batch, tokens, heads, kv_heads, dim;
    long page, pages, per_sequence;
    float scale, cap, offset;
    long window;
    const float *slopes;
} pam_hip_cache_shape;

/* The rotation (and norm) of pam_hip_rotary_fwd for the new tokens' queries and keys, a token's row of the tables being its place; q's go to q->y
 * (contiguous; padding's are zeros; q may be NULL), k's and, as they are, v's to their places in the cache.  A token whose place the table does not have, or whose
 * page is not there, is written nowhere.  Places of two tokens of a call must differ, and the cache shares no memory with what is read.  k->y, v->y and
 * v->weight are not read. */
int pam_hip_rotary_append(const pam_hip_heads *q, const pam_hip_heads *k, const pam_hip_heads *v, const float *cos, const float *sin,
                          long table_rows, float *cache_k, float *cache_v, long cache_sp, long cache_st, long cache_sh, long page,
                          long pages, long per_sequence, const int *table, const long long *lengths, const long long *counts,
                          long batch, long tokens, long dim, long rotated, int interleaved, float eps, float offset, void *stream);

/* The new tokens' queries (already in the cache are their keys and values, too) over the places 0 ... lengths + t of their sequences, or the last
 * `window` of those; scores, weights and results as above.  y [batch][tokens][heads][dim] is contiguous; padding's are zeros.  A place that the table does
 * not have, or on a page that is not there, makes the results that see it NaN. */
size_t pam_hip_cached_attention_workspace_bytes(const pam_hip_cache_shape *shape);
int pam_hip_cached_attention_fwd(const pam_hip_cache_shape *shape, const pam_hip_tokens *q, const float *cache_k, const float *cache_v,
                                 long cache_sp, long cache_st, long cache_sh, const int *pages, const long long *lengths,
                                 const long long *counts, float *y, void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* PAM_HIP_ATTENTION_H */

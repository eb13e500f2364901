/*
 * epure_paged.h -- C ABI of what lies between a served decoder layer's
 * packed linears: rotary positions, a paged key-value cache that is
 * quantised as it is written, and attention of new tokens over it.
 *
 * The reference leaves all of this to transformers (epure/runtime.py:373-415
 * builds a LlamaForCausalLM / Qwen3ForCausalLM and replaces its linears);
 * include/epure_decode.h covers it for one sequence with a contiguous f32
 * cache.  These entry points serve batches: sequences of any lengths share
 * one pool of pages.
 *
 * All entry points follow include/epure_hip.h conventions (device pointers,
 * caller-owned buffers, return codes, no host synchronisation, capture-safe).
 * The descriptors below are host structs, read before the call returns.
 *
 * Positions and page ids are read on the device, where nothing can raise:
 *   - a negative position marks a padded token: nothing is stored for it,
 *     and its output row is zeros;
 *   - a position past the tables (cos / sin rows, or the page table's
 *     width), or one whose page id lies outside [0, n_pages), stores
 *     nothing, and the output rows that need it are NaN.
 * No access leaves the buffers described, whatever they hold.
 *
 * A call of ep_rotate, ep_kv_append or ep_kv_read takes fewer than 2^32 lanes:
 * its rows (tokens times heads, of q, k and v together) times D / 16 rounded
 * up to a power of two.  One of more is declined.
 */
#ifndef EPURE_PAGED_H
#define EPURE_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "epure_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types of a cache, beside EP_F16 and EP_BF16 */
#define EP_E4M3 3 /* 8-bit float, 4 exponent bits, bias 7, largest value 448, no infinities */
#define EP_I8 4   /* signed 8-bit integer in [-127, 127] */

/* A [B, S, heads, D] tensor: strides in elements, each head's values adjacent. */
typedef struct {
    void *ptr;
    int dtype; /* EP_F32 / EP_F16 / EP_BF16 */
    int heads;
    int64_t stride_b, stride_s, stride_h;
} ep_heads;

/* The tokens of a call: position [B, S] of each and the pages of each sequence. */
typedef struct {
    int64_t B, S;
    const int64_t *positions;
    int64_t pos_stride_b, pos_stride_s;
    const int32_t *table; /* [B, width]: page of positions i * page .. i * page + page - 1 */
    int64_t table_stride, width;
} ep_tokens;

/*
 * The pool: k and v [n_pages][heads][page][D], dense, 16-byte aligned.  An
 * 8-bit row stands for code * scale, with scales [n_pages][heads][page] f32
 * (16-byte aligned; NULL for 16-bit types).  page: a power of two, 16..1024;
 * D: a multiple of 16, 16..256.
 */
typedef struct {
    void *k, *v;
    float *k_scale, *v_scale;
    int dtype; /* EP_F16 / EP_BF16 / EP_E4M3 / EP_I8 */
    int heads, page, D;
    int64_t n_pages;
} ep_kv_cache;

/*
 * A rotation: cos / sin [max_pos][dim / 2] f32, dense (an attention factor
 * is part of them).  dim: even; the first dim values of a head turn, the
 * rest is copied.  interleaved: pairs (2i, 2i + 1), else (i, i + dim / 2).
 */
typedef struct {
    const float *cos_t, *sin_t;
    int64_t max_pos;
    int dim, interleaved;
} ep_rotation;

/*
 * q_out, k_out [B, S, heads, D] (dense, the input's type) = q, k turned by
 * their positions: (a cos - b sin, b cos + a sin) in f32, each product
 * rounded before the sum, one rounding to the type at the end.  `inverse`
 * turns the other way: the gradient of the turn.  k->ptr may be NULL
 * (heads 0).  q and k have one type.  tokens->table is not read.
 */
int ep_rotate(const ep_heads *q, const ep_heads *k, const ep_rotation *rot, const ep_tokens *tokens, int64_t D,
              int inverse, void *q_out, void *k_out, void *stream);

/*
 * Stores the tokens' keys (turned where rot is given) and values in the
 * cache, and writes q turned to q_out [B, S, heads, D] (q may be NULL, with
 * or without rot).  The turned key enters the cache from f32, rounded once.
 *   16-bit types: rounded to the type.
 *   EP_I8: with m = max |x| of the row (at least 2^-100): scale = m / 127,
 *     code = rint(x * (127 / m)).
 *   EP_E4M3: scale = 2^e, the least e >= -100 with m <= 448 * 2^e; code =
 *     x / scale rounded to nearest even.
 *   A row that holds an infinity or a NaN: scale NaN, so that it reads back
 *   as NaN.
 * Two tokens of a call at one position of one sequence race.
 */
int ep_kv_append(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                 const ep_tokens *tokens, const ep_kv_cache *cache, void *q_out, void *stream);

/* k_out, v_out [B, S, heads, D] (dense, out_dtype) = the cache rows at the tokens' positions. */
int ep_kv_read(const ep_tokens *tokens, const ep_kv_cache *cache, void *k_out, void *v_out, int out_dtype,
               void *stream);

/*
 * out [B, S, q heads, D] (dense, q's type, 16-byte aligned): each token's
 * attention over the cache positions max(0, p - window + 1) .. p of its
 * sequence (window <= 0: from 0), p its own position, softmax of scale *
 * q . k; q heads a multiple of the cache's, head h reads cache head h / (q
 * heads / heads).  Tokens of a call may stand anywhere, in any order.  q:
 * EP_F16 or EP_BF16, 16-byte aligned with strides of whole 8 values; a 16-bit
 * cache has q's type; a table of at most 2^30 positions.  Scores, softmax and
 * sums are f32, the weights enter their product with 16 bits or more.  NaN
 * and infinities of positions that a token does not attend to do not reach
 * it; an infinite value that it attends to gives an infinity or NaN.  Up to
 * 2^31 - 1 query rows (tokens times query heads) are served, 2^30 - 1 of a
 * sequence on one cache head; more than 32 of those read the cache once per 32.
 * Workspace: ep_paged_attention_workspace() bytes (0 if the shape is
 * declined, or none is needed), 16-byte aligned, read and written by this call
 * alone.
 */
size_t ep_paged_attention_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache);
int ep_paged_attention(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, float scale,
                       int64_t window, void *out, void *workspace, size_t workspace_bytes, void *stream);

/*
 * The same attention for a batch whose tables begin with the same `shared`
 * pages (0 .. width; which row they are read from is not said): these pages are
 * computed once for the rows of the whole batch, then each sequence's own, and
 * the two are joined (a few pages are computed with the rest).  Every token's
 * position may lie in either.  At most 2^30 - 1 rows (tokens times query
 * heads) on one cache head.  Workspace: as above.
 */
size_t ep_paged_attention_shared_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                                           int64_t shared);
int ep_paged_attention_shared(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, int64_t shared,
                              float scale, int64_t window, void *out, void *workspace, size_t workspace_bytes,
                              void *stream);

/*
 * Bounds of the keys a cache holds: bounds [n_pages][heads][2][D] (dense,
 * 16-byte aligned; the cache's type, for 8-bit caches f32), the least and the
 * largest value of each column over a page's rows.  ep_kv_append_bounds stores
 * as ep_kv_append does; ep_kv_bounds takes the tokens as stored, behind an append
 * without a rotation.  Then each page that one of them lies on gets those of its rows from
 * 0 to the largest position of the call's tokens on it (a NaN among them is
 * both).  Sequences may have a page in common, and write it in one call: it
 * stands at one place of their tables then, as a page does that holds the keys
 * of some positions (where it stands at two, its bounds may be those of either).
 * Tokens that store nothing (past the rotation's or the page table, or on no page
 * of the pool) change nothing.
 */
int ep_kv_append_bounds(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                        const ep_tokens *tokens, const ep_kv_cache *cache, void *q_out, void *bounds, void *stream);
int ep_kv_bounds(const ep_tokens *tokens, const ep_kv_cache *cache, void *bounds, void *stream);

/*
 * blocks [B, S, q's cache heads, take] int32 (dense): for each token at position
 * p and each cache head the pages of the sequence (indices into its row of the
 * table, ascending, -1 behind the last) to attend to: page p / page, and of
 * those before it the take - 1 of the largest score
 *   sum_d hi_d sum_g max(q_gd, 0) + lo_d sum_g min(q_gd, 0),
 * g over the query heads of the cache head, in 64 bits; of equal scores the
 * lower page.  A score that is NaN, or of a page outside [0, n_pages), is above
 * all.  Tokens of negative positions and of positions past the table: all -1.
 * q: as in ep_paged_attention; its type need not be the cache's.  Workspace:
 * ep_kv_select_workspace() bytes, 16-byte aligned.
 */
size_t ep_kv_select_workspace(const ep_tokens *tokens, const ep_kv_cache *cache, int64_t take);
int ep_kv_select(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, const void *bounds, int64_t take,
                 int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream);

/*
 * ep_paged_attention over the pages that blocks [B, S, cache heads, take]
 * (int32, dense, take >= 1) names for each token and cache head, in any order:
 * the positions max(0, p - window + 1) .. p on them.  An index that is
 * negative, or not below the table's width, names none; one that is there
 * twice counts twice.  A token that sees no position gets zeros; one
 * that sees some, whose scores are all -inf, gets NaN as there.
 */
size_t ep_paged_attention_blocks_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                                           int64_t take);
int ep_paged_attention_blocks(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                              const int32_t *blocks, int64_t take, float scale, int64_t window, void *out,
                              void *workspace, size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* EPURE_PAGED_H */

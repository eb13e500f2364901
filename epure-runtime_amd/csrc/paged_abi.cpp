// extern "C" entry points of include/epure_paged.h: every check that the
// host can make, then the launch.  Kernels: paged.hip, attend.hip, select.hip.
#include <hip/hip_runtime.h>

#include "ep_internal.h"
#include "ep_paged.h"

using namespace ep;

namespace {

bool float_dtype(int dt) { return dt == EP_F32 || dt == EP_F16 || dt == EP_BF16; }
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

int check_heads(const char *what, const ep_heads *x, const ep_tokens *t)
{
    if (!x || x->heads < 1)
        return set_error(EP_ERR_ARG, "%s: no heads", what);
    if (!float_dtype(x->dtype))
        return set_error(EP_DECLINE_DTYPE, "%s: element type %d not served", what, x->dtype);
    if (t->B > 0 && t->S > 0 && !x->ptr)
        return set_error(EP_ERR_ARG, "%s: null pointer", what);
    return EP_OK;
}

int check_tokens(const ep_tokens *t, bool pages)
{
    if (!t || t->B < 0 || t->S < 0)
        return set_error(EP_ERR_ARG, "tokens: negative batch or length");
    const bool some = t->B > 0 && t->S > 0;
    if (t->B > 0 && t->S > (int64_t)0x7fffffff / t->B)
        return set_error(EP_DECLINE_SHAPE, "%lld x %lld tokens are more than one call takes", (long long)t->B,
                         (long long)t->S);
    if (some && !t->positions)
        return set_error(EP_ERR_ARG, "tokens: null positions");
    if (pages && (t->width < 0 || (some && t->width > 0 && !t->table)))
        return set_error(EP_ERR_ARG, "tokens: bad page table");
    return EP_OK;
}

int check_rotation(const ep_rotation *r, int64_t D)
{
    if (r->dim < 2 || r->dim % 2 || r->dim > D)
        return set_error(EP_ERR_ARG, "rotation of %d values in heads of %lld", r->dim, (long long)D);
    if (r->max_pos < 0 || (r->max_pos > 0 && (!r->cos_t || !r->sin_t)))
        return set_error(EP_ERR_ARG, "rotation: bad tables");
    return EP_OK;
}

int check_cache(const ep_kv_cache *c, PagedCache &out)
{
    if (!c || c->heads < 1 || c->n_pages < 1 || !c->k || !c->v)
        return set_error(EP_ERR_ARG, "cache: no pages, heads or storage");
    if (c->dtype != EP_F16 && c->dtype != EP_BF16 && c->dtype != EP_E4M3 && c->dtype != EP_I8)
        return set_error(EP_DECLINE_DTYPE, "cache element type %d not served", c->dtype);
    if (c->page < 16 || c->page > 1024 || (c->page & (c->page - 1)))
        return set_error(EP_DECLINE_SHAPE, "page of %d rows: a power of two from 16 to 1024 is served", c->page);
    if (c->D < 16 || c->D > 256 || c->D % 16)
        return set_error(EP_DECLINE_SHAPE, "heads of %d values: multiples of 16 up to 256 are served", c->D);
    const bool scaled = c->dtype == EP_E4M3 || c->dtype == EP_I8;
    if (scaled && (!c->k_scale || !c->v_scale))
        return set_error(EP_ERR_ARG, "cache: 8-bit rows need scales");
    if (!aligned16(c->k) || !aligned16(c->v) || (scaled && (!aligned16(c->k_scale) || !aligned16(c->v_scale))))
        return set_error(EP_ERR_ARG, "cache: storage must be 16-byte aligned");
    out = PagedCache{c->k, c->v, c->k_scale, c->v_scale, c->n_pages, c->dtype, c->heads, c->page,
                     __builtin_ctz((unsigned)c->page), c->D};
    return EP_OK;
}

PagedTokens tokens_of(const ep_tokens *t)
{
    return PagedTokens{t->positions, t->pos_stride_b, t->pos_stride_s, t->table, t->table_stride, t->width, t->B, t->S};
}

// Query rows over a cache, of any of the types that attention takes.
int check_query(const ep_heads *q, const ep_tokens *t, const ep_kv_cache *cache, PagedCache &c)
{
    int rc = check_tokens(t, true);
    if (rc == EP_OK)
        rc = check_heads("q", q, t);
    if (rc == EP_OK)
        rc = check_cache(cache, c);
    if (rc != EP_OK)
        return rc;
    if (t->width > 0x3fffffff >> c.page_shift)
        return set_error(EP_DECLINE_SHAPE, "a table of %lld pages of %d rows: up to 2^30 positions are served",
                         (long long)t->width, c.page);
    if (q->dtype == EP_F32)
        return set_error(EP_DECLINE_DTYPE, "attention: q must be f16 or bf16");
    if (q->heads % c.heads)
        return set_error(EP_ERR_ARG, "%d query heads over %d cache heads", q->heads, c.heads);
    if (!aligned16(q->ptr) || (t->B > 1 && q->stride_b % 8) || (t->S > 1 && q->stride_s % 8) ||
        (q->heads > 1 && q->stride_h % 8))
        return set_error(EP_DECLINE_SHAPE, "attention: q's heads must be 16-byte aligned");
    return EP_OK;
}

int check_attend(const ep_heads *q, const ep_tokens *t, const ep_kv_cache *cache, PagedCache &c)
{
    const int rc = check_query(q, t, cache, c);
    if (rc == EP_OK && (c.dtype == EP_F16 || c.dtype == EP_BF16) && c.dtype != q->dtype)
        return set_error(EP_DECLINE_DTYPE, "attention: a 16-bit cache must have q's type");
    return rc;
}

// Pages taken of a context: their positions fit 30 bits.
int check_take(int64_t take, const ep_tokens *t, const PagedCache &c)
{
    if (take < 1)
        return set_error(EP_ERR_ARG, "%lld pages a token", (long long)take);
    if (take > 0x3fffffff >> c.page_shift)
        return set_error(EP_DECLINE_SHAPE, "%lld pages of %d rows a token: up to 2^30 positions are served",
                         (long long)take, c.page);
    // rows times pages: the scores and lists of a call
    if (t->B * t->S > (INT64_MAX / 8) / ((int64_t)c.heads * (t->width > take ? t->width : take)))
        return set_error(EP_DECLINE_SHAPE, "lists of %lld pages are more than one call takes", (long long)take);
    return EP_OK;
}

int check_append(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                 const ep_tokens *tokens, const ep_kv_cache *cache, const void *q_out, PagedCache &c)
{
    int rc = check_tokens(tokens, true);
    if (rc == EP_OK)
        rc = check_heads("k", k, tokens);
    if (rc == EP_OK)
        rc = check_heads("v", v, tokens);
    if (rc == EP_OK && q)
        rc = check_heads("q", q, tokens);
    if (rc == EP_OK)
        rc = check_cache(cache, c);
    if (rc == EP_OK && rot)
        rc = check_rotation(rot, c.D);
    if (rc != EP_OK)
        return rc;
    if (k->dtype != v->dtype || (q && q->dtype != k->dtype))
        return set_error(EP_ERR_ARG, "append: q, k and v differ in type");
    if (k->heads != c.heads || v->heads != c.heads)
        return set_error(EP_ERR_ARG, "append: %d key and %d value heads for a cache of %d", k->heads, v->heads, c.heads);
    if (q && !q_out && tokens->B > 0 && tokens->S > 0)
        return set_error(EP_ERR_ARG, "append: null output");
    return EP_OK;
}

int check_bounds(const void *bounds)
{
    return bounds && aligned16(bounds) ? EP_OK : set_error(EP_ERR_ARG, "bounds must be 16-byte aligned storage");
}

}  // namespace

extern "C" {

int ep_rotate(const ep_heads *q, const ep_heads *k, const ep_rotation *rot, const ep_tokens *tokens, int64_t D,
              int inverse, void *q_out, void *k_out, void *stream)
{
    set_error(EP_OK, "");
    int rc = check_tokens(tokens, false);
    if (rc == EP_OK)
        rc = check_heads("q", q, tokens);
    const bool two = k && k->ptr;
    if (rc == EP_OK && two)
        rc = check_heads("k", k, tokens);
    if (rc != EP_OK)
        return rc;
    if (two && k->dtype != q->dtype)
        return set_error(EP_ERR_ARG, "rotation: q and k differ in type");
    if (!rot)
        return set_error(EP_ERR_ARG, "rotation: no tables");
    rc = check_rotation(rot, D);
    if (rc != EP_OK)
        return rc;
    if (D > 4096)
        return set_error(EP_DECLINE_SHAPE, "heads of %lld values: up to 4096 are served", (long long)D);
    if (tokens->B > 0 && tokens->S > 0 && (!q_out || (two && !k_out)))
        return set_error(EP_ERR_ARG, "rotation: null output");
    return launch_rotate(q, two ? k : nullptr, rot, tokens_of(tokens), D, inverse, q_out, k_out, (hipStream_t)stream);
}

int ep_kv_append(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                 const ep_tokens *tokens, const ep_kv_cache *cache, void *q_out, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    const int rc = check_append(q, k, v, rot, tokens, cache, q_out, c);
    return rc != EP_OK ? rc : launch_kv_append(q, k, v, rot, tokens_of(tokens), c, q_out, (hipStream_t)stream);
}

int ep_kv_append_bounds(const ep_heads *q, const ep_heads *k, const ep_heads *v, const ep_rotation *rot,
                        const ep_tokens *tokens, const ep_kv_cache *cache, void *q_out, void *bounds, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    int rc = check_append(q, k, v, rot, tokens, cache, q_out, c);
    if (rc == EP_OK)
        rc = check_bounds(bounds);
    if (rc != EP_OK)
        return rc;
    const PagedTokens tok = tokens_of(tokens);
    rc = launch_kv_append(q, k, v, rot, tok, c, q_out, (hipStream_t)stream);
    if (rc != EP_OK || tokens->B == 0 || tokens->S == 0)
        return rc;
    return launch_kv_bounds(tok, c, bounds, rot ? rot->max_pos : INT64_MAX, (hipStream_t)stream);
}

int ep_kv_read(const ep_tokens *tokens, const ep_kv_cache *cache, void *k_out, void *v_out, int out_dtype,
               void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    int rc = check_tokens(tokens, true);
    if (rc == EP_OK)
        rc = check_cache(cache, c);
    if (rc != EP_OK)
        return rc;
    if (!float_dtype(out_dtype))
        return set_error(EP_DECLINE_DTYPE, "cache read: element type %d not served", out_dtype);
    if (tokens->B > 0 && tokens->S > 0 && (!k_out || !v_out))
        return set_error(EP_ERR_ARG, "cache read: null output");
    return launch_kv_read(tokens_of(tokens), c, k_out, v_out, out_dtype, (hipStream_t)stream);
}

size_t ep_paged_attention_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache)
{
    set_error(EP_OK, "");
    PagedCache c;
    return check_attend(q, tokens, cache, c) == EP_OK ? attend_workspace(q, tokens_of(tokens), c) : 0;
}

int ep_paged_attention(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, float scale,
                       int64_t window, void *out, void *workspace, size_t workspace_bytes, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    const int rc = check_attend(q, tokens, cache, c);
    if (rc != EP_OK)
        return rc;
    if (tokens->B == 0 || tokens->S == 0)
        return EP_OK;
    if (!out)
        return set_error(EP_ERR_ARG, "attention: null output");
    if (!aligned16(out) || !aligned16(workspace))
        return set_error(EP_DECLINE_SHAPE, "attention: output and workspace must be 16-byte aligned");
    return launch_attend(q, tokens_of(tokens), c, scale, window, out, workspace, workspace_bytes, (hipStream_t)stream);
}

size_t ep_paged_attention_shared_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                                           int64_t shared)
{
    set_error(EP_OK, "");
    PagedCache c;
    if (check_attend(q, tokens, cache, c) != EP_OK || shared < 0 || shared > tokens->width)
        return 0;
    return attend_parts_workspace(q, tokens_of(tokens), c, shared);
}

int ep_paged_attention_shared(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, int64_t shared,
                              float scale, int64_t window, void *out, void *workspace, size_t workspace_bytes,
                              void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    const int rc = check_attend(q, tokens, cache, c);
    if (rc != EP_OK)
        return rc;
    if (shared < 0 || shared > tokens->width)
        return set_error(EP_ERR_ARG, "%lld shared pages in tables of %lld", (long long)shared, (long long)tokens->width);
    if (tokens->B == 0 || tokens->S == 0)
        return EP_OK;
    if (!out)
        return set_error(EP_ERR_ARG, "attention: null output");
    if (!aligned16(out) || !aligned16(workspace))
        return set_error(EP_DECLINE_SHAPE, "attention: output and workspace must be 16-byte aligned");
    return launch_attend_parts(q, tokens_of(tokens), c, shared, scale, window, out, workspace, workspace_bytes,
                               (hipStream_t)stream);
}

int ep_kv_bounds(const ep_tokens *tokens, const ep_kv_cache *cache, void *bounds, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    int rc = check_tokens(tokens, true);
    if (rc == EP_OK)
        rc = check_cache(cache, c);
    if (rc == EP_OK)
        rc = check_bounds(bounds);
    if (rc != EP_OK || tokens->B == 0 || tokens->S == 0)
        return rc;
    return launch_kv_bounds(tokens_of(tokens), c, bounds, INT64_MAX, (hipStream_t)stream);
}

size_t ep_kv_select_workspace(const ep_tokens *tokens, const ep_kv_cache *cache, int64_t take)
{
    set_error(EP_OK, "");
    PagedCache c;
    if (check_tokens(tokens, true) != EP_OK || check_cache(cache, c) != EP_OK || check_take(take, tokens, c) != EP_OK)
        return 0;
    return select_workspace(tokens_of(tokens), c, take);
}

int ep_kv_select(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache, const void *bounds, int64_t take,
                 int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    int rc = check_query(q, tokens, cache, c);
    if (rc == EP_OK)
        rc = check_take(take, tokens, c);
    if (rc == EP_OK)
        rc = check_bounds(bounds);
    if (rc != EP_OK || tokens->B == 0 || tokens->S == 0)
        return rc;
    if (!blocks)
        return set_error(EP_ERR_ARG, "select: null output");
    if (!aligned16(workspace))
        return set_error(EP_DECLINE_SHAPE, "select: the workspace must be 16-byte aligned");
    return launch_kv_select(q, tokens_of(tokens), c, bounds, take, blocks, workspace, workspace_bytes,
                            (hipStream_t)stream);
}

size_t ep_paged_attention_blocks_workspace(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                                           int64_t take)
{
    set_error(EP_OK, "");
    PagedCache c;
    if (check_attend(q, tokens, cache, c) != EP_OK || check_take(take, tokens, c) != EP_OK)
        return 0;
    return attend_blocks_workspace(q, tokens_of(tokens), c, take);
}

int ep_paged_attention_blocks(const ep_heads *q, const ep_tokens *tokens, const ep_kv_cache *cache,
                              const int32_t *blocks, int64_t take, float scale, int64_t window, void *out,
                              void *workspace, size_t workspace_bytes, void *stream)
{
    set_error(EP_OK, "");
    PagedCache c;
    int rc = check_attend(q, tokens, cache, c);
    if (rc == EP_OK)
        rc = check_take(take, tokens, c);
    if (rc != EP_OK)
        return rc;
    if (tokens->B == 0 || tokens->S == 0)
        return EP_OK;
    if (!out || !blocks)
        return set_error(EP_ERR_ARG, "attention: null output or list of pages");
    if (!aligned16(out) || !aligned16(workspace))
        return set_error(EP_DECLINE_SHAPE, "attention: output and workspace must be 16-byte aligned");
    return launch_attend_blocks(q, tokens_of(tokens), c, blocks, take, scale, window, out, workspace, workspace_bytes,
                                (hipStream_t)stream);
}

}  // extern "C"

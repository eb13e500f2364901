/*
 * epure_draft.h -- C ABI of the verification of drafted tokens: which of the
 * tokens that a cheaper model proposed a decoder's own probabilities let stand,
 * and the token that follows them.
 *
 * The reference decodes token by token (transformers' generate); there is no
 * counterpart.  Conventions of include/epure_hip.h: device pointers,
 * caller-owned buffers, return codes, no host synchronisation, capture-safe.
 */
#ifndef EPURE_DRAFT_H
#define EPURE_DRAFT_H

#include <stddef.h>
#include <stdint.h>

#include "epure_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Probabilities of B sequences: target [B][n + 1][V], and draft [B][n][V] or
 * NULL (the drafted tokens were certain: q = 1 for each, 0 elsewhere), both of
 * one type (EP_F32 / EP_F16 / EP_BF16), strides in elements, the values of one
 * step adjacent.  They need not sum to 1; a NaN or a negative one counts as 0.
 * drafted [B][n]: token ids; one outside [0, V) ends its sequence's draft.
 * uniforms [B][n + 1]: random numbers in [0, 1).
 */
typedef struct {
    int64_t B, V;
    int n, dtype;
    const void *target;
    int64_t target_stride_b, target_stride_s;
    const void *draft;
    int64_t draft_stride_b, draft_stride_s;
    const int64_t *drafted;
    int64_t drafted_stride_b, drafted_stride_s;
    const float *uniforms;
    int64_t uniforms_stride_b, uniforms_stride_s;
} ep_draft;

/*
 * accepted [B]: k, the number of drafted tokens ahead of the first with not
 * u_i q_i(x_i) < p_i(x_i).  tokens [B][n + 1]: those k, one token drawn, and -1
 * behind it.  That token is the first v for which
 *   sum over w <= v of r(w) > u_n * sum over all w of r(w),
 * r = max(p_k - q_k, 0) where a token was turned down (p_k, if that is zero
 * throughout), p_k where the draft ended; V - 1 if nothing weighs anything, the
 * last that weighs something if no sum passes (u_n >= 1).  Products and
 * sums are in 64 bits.  Workspace: ep_verify_draft_workspace() bytes, 16-byte
 * aligned, used by this call alone.
 */
size_t ep_verify_draft_workspace(const ep_draft *d);
int ep_verify_draft(const ep_draft *d, int64_t *accepted, int64_t *tokens, void *workspace, size_t workspace_bytes,
                    void *stream);

#ifdef __cplusplus
}
#endif

#endif /* EPURE_DRAFT_H */

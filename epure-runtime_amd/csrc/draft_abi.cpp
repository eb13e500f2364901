// extern "C" entry points of include/epure_draft.h: checks, then the launch.
// Kernels: draft.hip.
#include <hip/hip_runtime.h>

#include "ep_draft.h"
#include "ep_internal.h"
#include "epure_draft.h"

using namespace ep;

namespace {

int check_draft(const ep_draft *d)
{
    if (!d || d->B < 0 || d->n < 0 || d->V < 1)
        return set_error(EP_ERR_ARG, "verification: no vocabulary, or a negative size");
    if (d->dtype != EP_F32 && d->dtype != EP_F16 && d->dtype != EP_BF16)
        return set_error(EP_DECLINE_DTYPE, "verification: element type %d not served", d->dtype);
    if (d->n > 0x3fffffff || d->V > 0x7fffffff || d->B > 0x7fffffff)
        return set_error(EP_DECLINE_SHAPE, "verification: %lld sequences of %d drafted tokens over %lld",
                         (long long)d->B, d->n, (long long)d->V);
    if (d->B > 0 && (!d->target || !d->uniforms || (d->n > 0 && !d->drafted)))
        return set_error(EP_ERR_ARG, "verification: null pointer");
    return EP_OK;
}

}  // namespace

extern "C" {

size_t ep_verify_draft_workspace(const ep_draft *d)
{
    set_error(EP_OK, "");
    return check_draft(d) == EP_OK ? verify_workspace(d->B, d->V) : 0;
}

int ep_verify_draft(const ep_draft *d, int64_t *accepted, int64_t *tokens, void *workspace, size_t workspace_bytes,
                    void *stream)
{
    set_error(EP_OK, "");
    const int rc = check_draft(d);
    if (rc != EP_OK || d->B == 0)
        return rc;
    if (!accepted || !tokens)
        return set_error(EP_ERR_ARG, "verification: null output");
    if ((uintptr_t)workspace & 15)
        return set_error(EP_DECLINE_SHAPE, "verification: the workspace must be 16-byte aligned");
    const DraftTensors t{d->target, d->draft, d->target_stride_b, d->target_stride_s, d->draft_stride_b,
                         d->draft_stride_s, d->drafted, d->drafted_stride_b, d->drafted_stride_s, d->uniforms,
                         d->uniforms_stride_b, d->uniforms_stride_s, d->V, d->n};
    return launch_verify(t, d->B, d->dtype, accepted, tokens, workspace, workspace_bytes, (hipStream_t)stream);
}

}  // extern "C"

"""Verification of drafted tokens: which of the tokens that a cheaper model
proposed the decoder's own probabilities let stand, and the token that follows
them, on the gfx950 kernels (include/epure_draft.h).

The reference decodes token by token (transformers' generate).
"""
import ctypes

import torch

from .kernels import _abi
from .paged import _native, _require, _run


def verify_draft(target, drafted, uniforms, draft=None):
    """(accepted, tokens) of B sequences' drafted tokens.

    ``drafted`` ``[B, n]`` are token ids (int32 or int64; one outside the
    vocabulary ends its sequence's draft, so that ragged drafts are padded
    with -1), ``target`` ``[B, n + 1, V]`` the decoder's probabilities for each
    of them and for the token behind the last, ``draft`` ``[B, n, V]`` those
    they were drawn from, in the same type (float32, float16 or bfloat16).
    Without ``draft`` the proposals were certain (a lookup, a greedy model).
    Probabilities need not sum to 1; a NaN or a negative one counts as 0.
    ``uniforms`` ``[B, n + 1]`` are float32 random numbers in [0, 1).

    Token x of step i stands if ``uniforms[i] * draft[i, x] < target[i, x]``.
    The first that does not is replaced by one drawn from
    ``max(target[i] - draft[i], 0)``, and where all stand one more is drawn
    from the target: the first token at which the running sum of the weights
    exceeds ``uniforms[n]`` times their sum.  So drawn, the tokens are
    distributed as if the decoder had drawn each.  ``accepted`` ``[B]`` counts
    the drafted tokens that stand, ``tokens`` ``[B, n + 1]`` holds them, the
    one drawn, and -1 behind it (both int64).  Products and sums are in 64 bits.
    Nothing synchronizes, nothing is derived.  GPU tensors only."""
    call = _native()
    if call is not None:
        r = call.verify(target, drafted, uniforms, draft)
        if r is not NotImplemented:
            return r
    given = () if draft is None else (draft,)
    for t in (target, drafted, uniforms, *given):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"expected tensors, got {type(t).__name__}")
    _require(target, drafted, uniforms, *given)
    target, draft = target.detach(), None if draft is None else draft.detach()
    if _abi.dtype_code(target.dtype) is None:
        raise TypeError(f"probabilities must be float32, float16 or bfloat16, got {target.dtype}")
    if draft is not None and draft.dtype != target.dtype:
        raise TypeError(f"target is {target.dtype}, draft {draft.dtype}")
    if drafted.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"drafted tokens must be int32 or int64, got {drafted.dtype}")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"uniforms must be float32, got {uniforms.dtype}")
    if drafted.dim() != 2 or target.dim() != 3:
        raise ValueError(f"expected drafted [B, n] and target [B, n + 1, V], got {tuple(drafted.shape)} and "
                         f"{tuple(target.shape)}")
    (B, n), V = drafted.shape, target.shape[2]
    if tuple(target.shape) != (B, n + 1, V) or V < 1:
        raise ValueError(f"target {tuple(target.shape)} must be [{B}, {n + 1}, V]")
    if tuple(uniforms.shape) != (B, n + 1):
        raise ValueError(f"uniforms {tuple(uniforms.shape)} must be [{B}, {n + 1}]")
    if draft is not None and tuple(draft.shape) != (B, n, V):
        raise ValueError(f"draft {tuple(draft.shape)} must be [{B}, {n}, {V}]")
    drafted, uniforms = drafted.detach().to(torch.int64), uniforms.detach()
    target = target if target.stride(2) == 1 or V == 1 else target.contiguous()
    if draft is not None and draft.stride(2) != 1 and V > 1:
        draft = draft.contiguous()
    accepted = torch.empty(B, dtype=torch.int64, device=target.device)
    tokens = torch.empty(B, n + 1, dtype=torch.int64, device=target.device)
    if B == 0:
        return accepted, tokens
    some = draft is not None and n > 0
    d = _abi.Draft(B, V, n, _abi.dtype_code(target.dtype), target.data_ptr(), target.stride(0), target.stride(1),
                   draft.data_ptr() if some else None, draft.stride(0) if some else 0, draft.stride(1) if some else 0,
                   drafted.data_ptr() if n else None, drafted.stride(0), drafted.stride(1),
                   uniforms.data_ptr(), uniforms.stride(0), uniforms.stride(1))
    with torch.cuda.device(target.device):
        size = _abi.lib.ep_verify_draft_workspace(ctypes.byref(d))
        ws = torch.empty(size, dtype=torch.uint8, device=target.device)
        _run("ep_verify_draft", _abi.lib.ep_verify_draft(d, accepted.data_ptr(), tokens.data_ptr(), ws.data_ptr(), size,
                                                         _abi.stream_handle(target.device)))
    return accepted, tokens

"""The verification of drafted tokens off the GPU: the oracle against counted
outcomes, and what the entry points refuse before anything is launched."""
import ctypes

import pytest
import torch

import epure
from epure.kernels import _abi
from oracle import drafts as od
from oracle import paged as op

P = 64


@pytest.fixture(scope="module")
def lib():
    assert _abi._load() is not None, _abi.LOAD_ERROR
    return _abi.lib


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("certain", [False, True])
def test_verified_tokens_are_distributed_as_the_target(certain):
    """The first token of each of N runs: accepted or drawn anew, it has the
    target's distribution.  A count of expectation e deviates by less than 6
    sqrt(e) but for one run in 10^8."""
    g = torch.Generator().manual_seed(1)
    N, V = 20000, 5
    p = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05], dtype=torch.float64)
    q = torch.tensor([0.1, 0.5, 0.15, 0.05, 0.2], dtype=torch.float64)
    drafted = torch.full((N, 1), 1) if certain else torch.multinomial(q, N, True, generator=g)[:, None]
    u = torch.rand(N, 2, generator=g)
    _, tokens = od.verify(p.expand(N, 2, V), drafted, u, None if certain else q.expand(N, 1, V))
    count = torch.bincount(torch.tensor([t[0] for t in tokens]), minlength=V).double()
    assert ((count - N * p).abs() <= 6 * (N * p).sqrt()).all()


def test_selection_by_brute_force():
    """Score of a page: the largest over corners of its bounds of the sum of the group's q . k."""
    g = torch.Generator().manual_seed(2)
    lim = torch.randn(1, 9, 2, 2, 4, generator=g, dtype=torch.float64).sort(3).values
    q = torch.randn(1, 1, 6, 4, generator=g, dtype=torch.float64)
    got = op.select(q, lim, torch.tensor([[8 * 16]]), 16, 4)
    for h in range(2):
        best = []
        for j in range(8):
            lo, hi = lim[0, j, h]
            score = 0.0
            for x in q[0, 0, 3 * h:3 * h + 3]:
                score += max(sum(x[d] * (hi if c >> d & 1 else lo)[d] for d in range(4)).item() for c in range(16))
            best.append(score)
        assert got[0, 0, h].tolist() == sorted(sorted(range(8), key=lambda j: -best[j])[:3]) + [8]


# ------------------------------------------------------------------ refusals on the host
def draft(B=2, V=100, n=3, dtype=_abi.F32, target=P, drafted=P, uniforms=P):
    return _abi.Draft(B, V, n, dtype, target, V, V, None, 0, 0, drafted, n, 1, uniforms, n + 1, 1)


@pytest.mark.parametrize("bad,rc", [({"B": -1}, -1), ({"V": 0}, -1), ({"n": -1}, -1), ({"dtype": 7}, 1), ({"V": 1 << 40}, 2),
                                    ({"n": 1 << 30}, 2), ({"target": None}, -1), ({"drafted": None}, -1),
                                    ({"uniforms": None}, -1)])
def test_verification_refuses(lib, bad, rc):
    codes = {-1: "EP_ERR_ARG", 1: "EP_DECLINE_DTYPE", 2: "EP_DECLINE_SHAPE"}
    d = draft(**bad)
    got = lib.ep_verify_draft(ctypes.byref(d), P, P, P, 1 << 40, None)
    assert (got < 0) == (rc < 0) and got != 0, (codes[rc], got, _abi.last_error())
    assert _abi.last_error()
    if "target" not in bad:
        assert lib.ep_verify_draft_workspace(ctypes.byref(d)) == 0


def test_verification_wants_outputs_and_its_workspace(lib):
    d = draft()
    n = lib.ep_verify_draft_workspace(ctypes.byref(d))
    assert n > 0
    for out, tokens, ws, size in ((None, P, P, n), (P, None, P, n), (P, P, P + 8, n), (P, P, P, n - 1), (P, P, None, 0)):
        assert lib.ep_verify_draft(ctypes.byref(d), out, tokens, ws, size, None) != 0
    assert lib.ep_verify_draft(ctypes.byref(draft(B=0, target=None)), None, None, None, 0, None) == 0


def heads(n, d, ptr=P):
    return _abi.Heads(ptr, _abi.BF16, n, n * d, n * d, d)


def tokens(B=2, S=1, width=4):
    return _abi.Tokens(B, S, P, S, 1, P, width, width)


def cache(heads=2, D=64, dtype=_abi.BF16, page=16):
    return _abi.KVCache(P, P, None, None, dtype, heads, page, D, 4)


def test_paged_calls_refuse(lib):
    q, t, c = heads(4, 64), tokens(), cache()
    for shared in (-1, 5):
        assert lib.ep_paged_attention_shared(q, t, c, shared, 1.0, 0, P, P, 1 << 40, None) < 0
        assert lib.ep_paged_attention_shared_workspace(q, t, c, shared) == 0
    large = cache(page=1024)
    assert lib.ep_paged_attention_shared_workspace(q, t, large, 2) > 0
    assert lib.ep_paged_attention_shared(q, t, large, 2, 1.0, 0, P, None, 0, None) < 0
    assert "workspace" in _abi.last_error()
    assert lib.ep_paged_attention_blocks(q, t, c, None, 2, 1.0, 0, P, P, 1 << 40, None) < 0
    for take in (0, -1, 1 << 27):
        assert lib.ep_paged_attention_blocks(q, t, c, P, take, 1.0, 0, P, P, 1 << 40, None) != 0
        assert lib.ep_kv_select(q, t, c, P, take, P, P, 1 << 60, None) != 0
    assert lib.ep_kv_select(q, t, c, None, 2, P, P, 1 << 40, None) < 0
    assert lib.ep_kv_select(q, t, c, P + 8, 2, P, P, 1 << 40, None) < 0
    assert lib.ep_kv_select(q, t, c, P, 2, None, P, 1 << 40, None) < 0
    assert lib.ep_kv_select(q, tokens(width=600), c, P, 2, P, None, 0, None) != 0
    long = tokens(width=600)          # few pages, or all: no scores in memory
    assert lib.ep_kv_select_workspace(t, c, 3) == lib.ep_kv_select_workspace(long, c, 600) == 0
    assert lib.ep_kv_select_workspace(long, c, 1) == 0 < lib.ep_kv_select_workspace(long, c, 2)
    assert lib.ep_kv_select(heads(3, 64), t, c, P, 2, P, P, 1 << 40, None) < 0
    assert lib.ep_kv_bounds(t, c, None, None) < 0 and lib.ep_kv_bounds(t, c, P + 4, None) < 0
    many = tokens(B=1 << 15, S=1 << 15, width=1 << 20)
    for rc in (lib.ep_kv_select(q, many, c, P, 2, P, P, 1 << 62, None),
               lib.ep_paged_attention_shared(q, many, c, 2, 1.0, 0, P, P, 1 << 62, None),
               lib.ep_paged_attention_blocks(q, many, c, P, 2, 1.0, 0, P, P, 1 << 62, None),
               lib.ep_kv_bounds(tokens(B=1 << 30, S=1), cache(heads=4), P, None)):
        assert rc > 0 and "more than one call" in _abi.last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the refusal without a GPU")
def test_host_tensors_are_refused():
    t = torch.full((1, 2, 4), 0.25)
    with pytest.raises(RuntimeError, match="not available"):
        epure.verify_draft(t, torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))
    c = epure.PagedKVCache(2, 16, 1, 16, device="cpu", bounds=True)
    q, pos, table = torch.zeros(1, 1, 1, 16), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="not available"):
        c.select(q, pos, table, 1)
    with pytest.raises(RuntimeError, match="not available"):
        c.attend(q, pos, table, shared=1)


def test_native_calls_leave_host_tensors_to_the_python_path():
    assert _abi._load() is not None and _abi.call is not None, (_abi.LOAD_ERROR, _abi.CALL_ERROR)
    x, pos = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int64)
    table, c = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    lim, b, call = c[:, :, :2].contiguous(), torch.zeros(1, 1, 1, 1, dtype=torch.int32), _abi.call
    assert call.select(x, pos, table, 1, c, c, None, None, lim) is NotImplemented
    assert call.attend_more(x, pos, table, None, None, 1, None, c, c, None, None) is NotImplemented
    assert call.attend_more(x, pos, table, None, None, 0, b, c, c, None, None) is NotImplemented
    assert call.append_bounds(x, x, pos, table, None, None, None, False, c, c, None, None, lim) is NotImplemented
    assert call.verify(torch.zeros(1, 2, 4), pos, torch.zeros(1, 2), None) is NotImplemented
    for f in (call.select, call.attend_more, call.append_bounds, call.verify):
        with pytest.raises(TypeError):
            f(x)

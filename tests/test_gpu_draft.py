"""Verification of drafted tokens on the GPU against oracle/drafts.py."""
import pytest
import torch

import epure
from epure.kernels import _abi, cuda
from oracle import drafts as od

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def made(g, B, n, V, dtype, near=0.3, std=2.0):
    """Probabilities of both models, tokens that the draft would draw, uniforms."""
    logits = torch.randn(B, n + 1, V, generator=g, device=DEV) * std
    target = torch.softmax(logits, -1).to(dtype)
    draft = torch.softmax(logits[:, :n] + near * torch.randn(B, n, V, generator=g, device=DEV), -1)
    drafted = torch.multinomial(draft.view(B * n, V), 1, generator=g).view(B, n) if n else \
        torch.zeros(B, 0, dtype=torch.int64, device=DEV)
    return target, drafted, torch.rand(B, n + 1, generator=g, device=DEV), draft.to(dtype)


def same(got, want):
    assert got[0].dtype == got[1].dtype == torch.int64
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,n,V", [(41, 2, 51201), (1050, 1, 1500), (700, 2, 3077), (3, 1, 1024), (2, 2, 1025)])
def test_verification_of_more_pieces_than_workgroups_at_once(B, n, V, dtype):
    """Rows of 51, 2, 4 and, for one workgroup each, 1 and 2 pieces."""
    g = gen(B + V)
    target, drafted, u, draft = made(g, B, n, V, dtype)
    same(epure.verify_draft(target, drafted, u, draft=draft), od.verify(target, drafted, u, draft))
    same(epure.verify_draft(target, drafted, u), od.verify(target, drafted, u))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,n,V", [(1, 1, 1), (1, 1, 2), (3, 4, 1000), (2, 2, 4096), (2, 3, 4097), (5, 1, 8191), (70, 5, 63),
                                   (1, 70, 300), (2, 4, 20001)])
def test_verification(B, n, V, dtype):
    g = gen(B + V)
    target, drafted, u, draft = made(g, B, n, V, dtype)
    same(epure.verify_draft(target, drafted, u, draft=draft), od.verify(target, drafted, u, draft))
    same(epure.verify_draft(target, drafted, u), od.verify(target, drafted, u))
    drafted[torch.rand(B, n, generator=g, device=DEV) < 0.2] = -1            # drafts that end earlier
    drafted[B - 1, n - 1] = V
    same(epure.verify_draft(target, drafted, u, draft=draft), od.verify(target, drafted, u, draft))
    same(epure.verify_draft(target, drafted.int(), u), od.verify(target, drafted, u))


def test_without_a_draft_a_token_is_drawn():
    g = gen(1)
    target, drafted, u, draft = made(g, 4, 0, 777, F32)
    got = epure.verify_draft(target, drafted, u)
    same(got, od.verify(target, drafted, u))
    assert got[1].shape == (4, 1) and (got[0] == 0).all()
    same(epure.verify_draft(target, drafted, u, draft=draft), od.verify(target, drafted, u))


def test_borders_are_exact():
    """u q = p does not stand; a goal that a running sum reaches is not passed; u = 0 takes the first weight."""
    p = torch.full((1, 2, 8), 0.125, device=DEV)
    q = torch.full((1, 1, 8), 0.25, device=DEV)
    x = torch.tensor([[3]], device=DEV)
    for u0, k in ((0.5, 0), (0.49999997, 1)):
        for u1 in (0.0, 0.125, 0.5, 0.875, 0.99999994):
            u = torch.tensor([[u0, u1]], device=DEV)
            got = epure.verify_draft(p, x, u, draft=q)
            same(got, od.verify(p, x, u, q))
            assert got[0].item() == k and got[1][0, k].item() == int(u1 * 8)
    zero = torch.zeros(1, 1, 8, device=DEV)
    same(epure.verify_draft(p, x, torch.zeros(1, 2, device=DEV), draft=zero), ([1], [[3, 0]]))
    p[0, 0, 3] = 0.0            # 0 < 0 is false
    same(epure.verify_draft(p, x, torch.zeros(1, 2, device=DEV), draft=zero), ([0], [[0, -1]]))


def test_weights_that_are_nothing_or_not_numbers():
    V = 5000
    x, u = torch.tensor([[2]], device=DEV), torch.tensor([[0.9, 0.5]], device=DEV)
    p = torch.zeros(1, 2, V, device=DEV)
    same(epure.verify_draft(p, x, u), ([0], [[V - 1, -1]]))                    # nothing weighs anything
    p[0, 0, 4500] = 1.0
    same(epure.verify_draft(p, x, u, draft=p[:, :1]), ([0], [[4500, -1]]))     # nothing is left of p - q
    p[0, 0, 10], p[0, 0, 11] = float("nan"), -3.0
    same(epure.verify_draft(p, x, u), ([0], [[4500, -1]]))
    for bad in (1.0, 2.0, float("nan"), float("inf")):
        u[0, 1] = bad
        same(epure.verify_draft(p, x, u), ([0], [[4500, -1]]))
    u[0, 1] = -1.0
    p[0, 0, 20] = 1e-30
    same(epure.verify_draft(p, x, u), ([0], [[20, -1]]))
    u[0] = float("nan")
    same(epure.verify_draft(p, x, u), ([0], [[4500, -1]]))


def test_strides_streams_graphs_and_the_python_path(monkeypatch):
    g = gen(3)
    target, drafted, u, draft = made(g, 3, 4, 5001, F16)
    want = od.verify(target, drafted, u, draft)
    t2 = torch.empty(5, 3, 5003, dtype=F16, device=DEV)
    t2[:, :, 1:5002] = target.transpose(0, 1)
    flipped = target.transpose(1, 2).contiguous().transpose(1, 2)
    d2 = torch.stack((drafted, drafted), -1)[..., 0]
    u2 = u.T.contiguous().T
    q2 = draft.transpose(1, 2).contiguous().transpose(1, 2)
    for t in (target, t2[:, :, 1:5002].transpose(0, 1), flipped):
        for x, v, q in ((drafted, u, draft), (d2, u2, q2)):
            same(epure.verify_draft(t, x, v, draft=q), want)
    one = draft[:1, :1].expand(3, 4, 5001)
    same(epure.verify_draft(target, drafted, u, draft=one), od.verify(target, drafted, u, one))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = epure.verify_draft(target, drafted, u, draft=draft)
    torch.cuda.current_stream().wait_stream(side)
    same(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = epure.verify_draft(target, drafted, u, draft=draft)
    for _ in range(3):
        for a, b in zip((target, drafted, u, draft), made(g, 3, 4, 5001, F16)):
            a.copy_(b)
        eager = epure.verify_draft(target, drafted, u, draft=draft)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        same(out, od.verify(target, drafted, u, draft))
    monkeypatch.setattr(_abi, "call", None)
    same(epure.verify_draft(target, drafted, u, draft=draft), od.verify(target, drafted, u, draft))


def test_refusals():
    g = gen(4)
    target, drafted, u, draft = made(g, 2, 3, 50, F32)
    for bad, error in (((target.double(), drafted, u), TypeError), ((target, drafted.float(), u), TypeError),
                       ((target, drafted, u.double()), TypeError), ((target[:, :3], drafted, u), ValueError),
                       ((target, drafted, u[:, :3]), ValueError), ((target, drafted[0], u), ValueError),
                       ((target[..., :0], drafted, u), ValueError), ((target.cpu(), drafted, u), ValueError),
                       ((target, drafted.tolist(), u), TypeError), ((target, drafted, u, draft.half()), TypeError),
                       ((target, drafted, u, draft[..., :49]), ValueError), ((target, drafted, u, draft[:, :2]), ValueError)):
        with pytest.raises(error):
            epure.verify_draft(*bad)
    a, b = epure.verify_draft(target[:0], drafted[:0], u[:0])
    assert a.shape == (0,) and b.shape == (0, 4)
    got = epure.verify_draft(target.requires_grad_(), drafted, u)
    assert not got[0].requires_grad

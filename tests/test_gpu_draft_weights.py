"""Probabilities that are negative or no numbers count as zeros, the target's
and the draft's."""
import pytest
import torch

import epure
from epure.kernels import cuda
from oracle import drafts as od
from test_gpu_draft import BF16, DEV, F16, F32, gen, made, same

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def cleaned(t):
    """What such values count as, exactly."""
    return torch.where(t > 0, t, 0.0)


def test_a_negative_draft_adds_nothing_and_one_that_is_no_number_takes_nothing():
    V = 8
    p = torch.zeros(1, 2, V, device=DEV)
    q = torch.zeros(1, 1, V, device=DEV)
    p[0, 0, :4] = torch.tensor([0.25, 0.25, 0.25, 0.25], device=DEV)
    q[0, 0, :4] = torch.tensor([0.5, -8.0, NAN, 0.25], device=DEV)        # left: 0, 0.25, 0.25, 0
    x = torch.tensor([[0]], device=DEV)
    for u, want in ((0.0, 1), (0.49, 1), (0.5, 2), (0.9999, 2)):
        got = epure.verify_draft(p, x, torch.tensor([[0.75, u]], device=DEV), draft=q)
        same(got, ([0], [[want, -1]]))
        same(got, od.verify(p, x, torch.tensor([[0.75, u]]), q))
    p[0, 0, 5], q[0, 0, 5] = -1.0, -4.0              # nothing, though -1 - -4 is positive
    same(epure.verify_draft(p, x, torch.tensor([[0.75, 0.9999]], device=DEV), draft=q), ([0], [[2, -1]]))
    for bad, k in ((5, 0), (2, 1), (1, 1), (3, 1)):          # 0 < 0; 0 < 0.25; 0 < 0.25; 0.75 * 0.25 < 0.25
        u = torch.tensor([[0.75, 0.0]], device=DEV)
        y = torch.tensor([[bad]], device=DEV)
        got = epure.verify_draft(p, y, u, draft=q)
        assert got[0].item() == k
        same(got, od.verify(p, y, u, q))


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,n,V", [(3, 4, 1000), (2, 3, 4097), (700, 2, 3077)])
def test_as_zeros_in_their_place(B, n, V, dtype):
    g = gen(B + V)
    target, drafted, u, draft = made(g, B, n, V, dtype)
    for t in (target, draft):
        r = torch.rand(t.shape, generator=g, device=DEV)
        t[r < 0.1] = NAN
        t[(r > 0.1) & (r < 0.3)] = -0.5
        bits, signalling = {F32: (torch.int32, 0x7f800001), F16: (torch.int16, 0x7c01), BF16: (torch.int16, 0x7f81)}[dtype]
        t.view(bits)[(r > 0.3) & (r < 0.35)] = signalling
    if B * n > 3:
        drafted.view(-1)[3] = -1
    got = epure.verify_draft(target, drafted, u, draft=draft)
    want = epure.verify_draft(cleaned(target), drafted, u, draft=cleaned(draft))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    if B < 100:
        same(got, od.verify(target, drafted, u, draft))
        same(epure.verify_draft(target, drafted, u), od.verify(target, drafted, u))

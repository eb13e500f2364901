"""Attention behind shared pages, against the oracle's attention over each
whole context: the same results as without sharing."""
import pytest
import torch

import epure
from epure.kernels import cuda
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=BF16, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def tables(g, B, shared, own, spare=2):
    """Tables [B, shared + own] that begin with the same pages, pages in any order."""
    ids = torch.randperm(shared + B * own + spare, generator=g, device=DEV).to(torch.int32)
    return torch.cat((ids[:shared].expand(B, shared), ids[shared:shared + B * own].view(B, own)), 1).contiguous()


def filled(g, B, shared, own, page, heads, D, dtype):
    cache = epure.PagedKVCache(shared + B * own + 2, page, heads, D, dtype, DEV)
    table = tables(g, B, shared, own)
    L = (shared + own) * page
    xdt = dtype if dtype.itemsize == 2 else BF16
    k, v = normal(g, B, L, heads, D, dtype=xdt), normal(g, B, L, heads, D, dtype=xdt)
    k[:, :shared * page], v[:, :shared * page] = k[:1, :shared * page], v[:1, :shared * page]
    cache.append(k, v, torch.arange(L, device=DEV), table)
    return (cache, table, *cache.read(torch.arange(L, device=DEV).expand(B, L), table, F32))


def check(got, q, k, v, pos, scale, window=None):
    out, mag, big = op.attend(q, k, v, pos, scale, window)
    assert torch.equal(got.cpu().isnan(), out.isnan())
    ok = ~out.isnan()
    tol = op.attend_tolerance(out, mag, big, got.dtype, q.shape[-1])
    bad = (got.cpu().double() - out).abs()[ok] > tol[ok]
    assert not bad.any(), f"{bad.sum().item()} of {bad.numel()} off"


CASES = [  # B, S, shared (1024 positions or more), own, page, G, heads, D
    (2, 1, 64, 1, 16, 1, 1, 64), (3, 1, 65, 3, 16, 4, 2, 128), (5, 1, 34, 1, 32, 2, 1, 96), (2, 5, 66, 2, 16, 5, 2, 80),
    (9, 3, 67, 2, 16, 3, 1, 48), (40, 1, 64, 1, 16, 2, 2, 16), (3, 1, 17, 9, 64, 8, 1, 192), (2, 2, 70, 1, 16, 20, 1, 256),
    (17, 1, 40, 1, 32, 4, 1, 128), (6, 8, 33, 2, 32, 3, 1, 144), (20, 2, 65, 1, 16, 1, 2, 160), (2, 1, 9, 2, 128, 1, 3, 112),
    (2, 1, 1, 1, 1024, 2, 1, 32), (3, 2, 5, 2, 16, 2, 1, 64)]


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,shared,own,page,G,heads,D", CASES)
def test_shared_pages(B, S, shared, own, page, G, heads, D, dtype):
    """Positions in the shared pages, behind them, at both ends, padded and past the table."""
    g = gen(B * D + S)
    cache, table, k, v = filled(g, B, shared, own, page, heads, D, dtype)
    q = normal(g, B, S, G * heads, D, dtype=dtype if dtype.itemsize == 2 else F16 if D % 48 == 0 else BF16, std=2.0)
    P, L = shared * page, (shared + own) * page
    pos = torch.randint(0, L, (B, S), generator=g, device=DEV)
    edge = torch.tensor([P - 1, P, L - 1, 0, -1, L, P + 1], device=DEV)
    pos.view(-1)[:min(7, B * S)] = edge[:min(7, B * S)]
    for window in (None, 17, 1024, 1029, P + 3):
        check(cache.attend(q, pos, table, window=window, shared=shared), q, k, v, pos, D ** -0.5, window)
    check(cache.attend(q, pos, table, scale=0.3, shared=shared - 1), q, k, v, pos, 0.3)


def test_all_pages_shared_and_none():
    g = gen(2)
    cache, table, k, v = filled(g, 4, 70, 1, 16, 2, 64, BF16)
    q, pos = normal(g, 4, 1, 4, 64, std=2.0), torch.tensor([[1119], [3], [1040], [-1]], device=DEV)
    check(cache.attend(q, pos, table[:, :70], shared=70), q, k[:, :1120], v[:, :1120], pos, 0.125)
    assert torch.equal(cache.attend(q, pos, table, shared=0), cache.attend(q, pos, table))
    # one sequence shares with nobody
    assert torch.equal(cache.attend(q[:1], pos[:1], table[:1], shared=70), cache.attend(q[:1], pos[:1], table[:1]))


@pytest.mark.parametrize("dtype", [BF16, I8])
def test_pages_that_the_pool_lacks_and_values_that_are_not_finite(dtype):
    """A missing page is a NaN to who sees a position on it; so is a value that is not finite, and to nobody else."""
    g = gen(3)
    at = 63 * 16
    cache, table, k, v = filled(g, 40, 67, 2, 16, 1, 64, dtype)
    q = normal(g, 40, 1, 2, 64, std=2.0)
    pos = (torch.arange(40, device=DEV) * 2 + 16)[:, None] + at    # 16 .. 94 behind 1008
    table[:, 65] = 1 << 20           # positions 32 .. 47, shared
    table[20, 67] = -1               # 64 .. 79 of sequence 20 (position 56: not seen), 30 (76: seen)
    table[30, 67] = -1
    got = cache.attend(q, pos, table, shared=67)
    want = ((pos >= at + 32) | (torch.arange(40, device=DEV)[:, None] == 30))[..., None, None].expand_as(got)
    assert torch.equal(got.isnan(), want)
    for window in (5, 1030):
        assert torch.equal(cache.attend(q, pos, table, shared=67, window=window).isnan()[:, 0, 0, 0].cpu(), torch.tensor(
            [any(32 <= j - at < 48 or (i == 30 and 64 <= j - at < 80) for j in range(max(p - window + 1, 0), p + 1))
             for i, p in enumerate(pos[:, 0].tolist())]))
    cache, table, k, v = filled(g, 40, 67, 2, 16, 1, 64, dtype)
    page, row = int(table[0, 64]), 5                                # position 1029
    if dtype == BF16:
        cache.v[page, 0, row, 7] = float("inf")
        cache.k[page, 0, row + 1] = float("nan")
    else:
        cache.v_scale[page, 0, row] = float("inf")
        cache.k_scale[page, 0, row + 1] = float("nan")
    got = cache.attend(q, pos, table, shared=67)
    assert not got[:3].isnan().any() and not got[:3].isinf().any()          # positions 1024, 1026, 1028
    assert got[3:].isnan().any(-1).all()


def test_strided_queries_and_other_streams_and_graphs():
    g = gen(4)
    cache, table, k, v = filled(g, 6, 66, 2, 16, 2, 128, BF16)
    q = normal(g, 6, 2, 8, 128, std=2.0)
    pos = torch.randint(0, 68 * 16, (6, 2), generator=g, device=DEV)
    want = cache.attend(q, pos, table, shared=66)
    check(want, q, k, v, pos, 128 ** -0.5)
    wide = torch.empty(6, 2, 8, 136, dtype=BF16, device=DEV)
    wide[..., :128] = q
    odd = torch.empty(6 * 2 * 8 * 128 + 1, dtype=BF16, device=DEV)[1:].view(6, 2, 8, 128)
    odd.copy_(q)
    for x in (wide[..., :128], odd, q.transpose(0, 1).contiguous().transpose(0, 1),
              q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(cache.attend(x, pos, table, shared=66), want)
    assert torch.equal(cache.attend(q, pos.T.contiguous().T, torch.cat((table, table), 1)[:, :68], shared=66), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(q, pos, table, shared=66)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, pos, table, shared=66)
    for i in range(3):
        pos.copy_(torch.randint(-1, 68 * 16 + 1, (6, 2), generator=g, device=DEV))
        q.copy_(normal(g, 6, 2, 8, 128, std=2.0))
        want = cache.attend(q, pos, table, shared=66)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.nan_to_num(7.0), want.nan_to_num(7.0))


def test_refusals():
    g = gen(5)
    cache, table, *_ = filled(g, 2, 2, 1, 16, 1, 64, BF16)
    q, pos = normal(g, 2, 1, 1, 64), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    blocks = torch.zeros(2, 1, 1, 2, dtype=torch.int32, device=DEV)
    for bad, error in (({"shared": 4}, ValueError), ({"shared": -1}, ValueError), ({"shared": 1.5}, TypeError),
                       ({"shared": 1, "blocks": blocks}, ValueError), ({"shared": 1, "window": 0}, ValueError)):
        with pytest.raises(error):
            cache.attend(q, pos, table, **bad)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.attend(q.requires_grad_(), pos, table, shared=1)
    assert cache.attend(q.detach()[:0], pos[:0], table[:0], shared=1).shape == (0, 1, 1, 64)

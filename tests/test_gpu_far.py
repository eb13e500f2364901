"""Shared and selected pages, their bounds and drafted tokens far into large
tensors, and through strides: the same bits as near the beginning of small ones."""
import pytest
import torch

import epure
from epure.kernels import cuda
from test_gpu_shared import BF16, DEV, F16, I8, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("B,G", [(2, 4), (12, 4), (2, 17), (2, 34)])
def test_pages_past_four_gib(B, G, dtype):
    """Units, rows through LDS with the others beside them and behind them; bounds, scores, lists."""
    heads, D, page, shared, own = 4, 128, 16, 600, 9
    used = shared + B * own
    far = 2 ** 32 // dtype.itemsize // (page * heads * D) + 5
    near = torch.empty(B, shared + own, dtype=torch.int32, device=DEV)
    near[:, :shared] = torch.arange(shared, device=DEV)
    near[:, shared:] = torch.arange(shared, used, device=DEV).view(B, own)
    P, L = shared * page, own * page
    got = []
    for at in (0, far):
        g = gen(B + G)
        cache = epure.PagedKVCache(at + used, page, heads, D, dtype, DEV, bounds=True)
        table = near + at
        k, v = (normal(g, 1, P, heads, D) for _ in range(2))
        cache.append(k, v, torch.arange(P, device=DEV)[None], table[:1])
        k, v = (normal(g, B, L, heads, D) for _ in range(2))
        cache.append(k, v, (P + torch.arange(L, device=DEV)).expand(B, L), table)
        q = normal(g, B, 1, G * heads, D, std=2.0)
        pos = torch.randint(P, P + L, (B, 1), generator=g, device=DEV)
        blocks = cache.select(q, pos, table, 40)
        got.append([cache.k_bounds[table.long()], blocks, cache.attend(q, pos, table, blocks=blocks),
                    cache.attend(q, pos, table, shared=shared)])
        del cache
    for a, b in zip(*got):
        assert torch.equal(a, b) and a.isfinite().all()


def test_probabilities_past_four_gib():
    n, V = 7, 128256
    B = 2 ** 31 // ((n + 1) * V) + 9
    g = gen(1)
    target, draft = torch.zeros(B, n + 1, V, dtype=F16, device=DEV), torch.zeros(B, n, V, dtype=F16, device=DEV)
    drafted = torch.randint(0, V, (B, n), generator=g, device=DEV)
    u = torch.rand(B, n + 1, generator=g, device=DEV)
    for t in (target, draft):
        t[-5:] = torch.rand(5, t.shape[1], V, generator=g, device=DEV)
    got = epure.verify_draft(target, drafted, u, draft=draft)
    want = epure.verify_draft(target[-5:].clone(), drafted[-5:], u[-5:], draft=draft[-5:].clone())
    assert torch.equal(got[0][-5:], want[0]) and torch.equal(got[1][-5:], want[1])
    assert (got[0][:-5] == 0).all() and (got[1][:-5, 0] == V - 1).all()      # nothing weighs anything


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("B,S,G", [(40, 1, 2), (9, 4, 8), (5, 5, 8)])
def test_strides(B, S, G, dtype):
    """Queries among keys and values, a table in a wider one, positions of one row for all: as of their copies."""
    heads, D, page, shared, own = 8, 96, 32, 330, 2
    g = gen(B + S)
    cache = epure.PagedKVCache(shared + B * own, page, heads, D, dtype, DEV)
    wide = torch.full((2 * B, shared + own + 7), -1, dtype=torch.int32, device=DEV)
    table = wide[::2, 3:3 + shared + own]
    table[:, :shared] = torch.arange(shared, device=DEV)
    table[:, shared:] = torch.arange(shared, shared + B * own, device=DEV).view(B, own)
    for pool in (cache.k, cache.v):
        pool.copy_((torch.randn(pool.shape, generator=g, device=DEV) * (30.0 if dtype == I8 else 1.0)).to(dtype))
    if dtype == I8:
        cache.k_scale.fill_(0.03)
        cache.v_scale.fill_(0.03)
    q = normal(g, S, B, (G + 2) * heads, D, std=2.0).transpose(0, 1)[:, :, heads:(G + 1) * heads]
    pos = torch.arange(shared * page + 3, shared * page + 3 + S, device=DEV)[None].expand(B, S)
    got = cache.attend(q, pos, table, shared=shared)
    assert torch.equal(got, cache.attend(q.contiguous(), pos.contiguous(), table.contiguous(), shared=shared))
    one = torch.cat([cache.attend(q[b:b + 1], pos[:1], table[b:b + 1]) for b in range(B)])
    # two roundings to bf16 (2^-8 between them) of sums of weights that add up to 1 over values of 4 and 2^-16 each
    assert ((got.float() - one.float()).abs() <= 2.0 ** -6 * one.float().abs() + 2.0 ** -9).all()

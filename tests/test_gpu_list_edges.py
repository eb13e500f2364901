"""Attention over a list of pages: a token whose scores are all -inf gets NaN,
as without a list; only one that sees no position gets zeros."""
import pytest
import torch

import epure
from epure.kernels import cuda
from test_gpu_select import BF16, DEV, F16, check, filled, gen, normal

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("width,page,G,take", [(4, 16, 2, 3), (40, 16, 5, 40), (5, 1024, 1, 3), (130, 32, 17, 128)])
def test_scores_of_minus_infinity(width, page, G, take, dtype):
    """One piece a list and several (those of the last two): every key seen is -inf in a column where q is positive."""
    g = gen(width)
    cache, table, k, v = filled(g, 2, width, page, 1, 64, dtype)
    q = normal(g, 2, 1, G, 64, dtype=dtype)
    q[..., 7] = 1.0
    L = width * page
    pos = torch.tensor([[L - 1], [L - page - 3]], device=DEV)
    blocks = torch.arange(take, dtype=torch.int32, device=DEV).flip(0).expand(2, 1, 1, take).contiguous()
    blocks[1, 0, 0, 0] = -1
    plain = cache.attend(q, pos, table, blocks=blocks)
    check(plain, q, k, v, pos, blocks, page, 0.125)
    held = cache.k.clone()
    cache.k[..., 7] = -INF
    got = cache.attend(q, pos, table, blocks=blocks)
    assert got.isnan().all()
    assert cache.attend(q, pos, table).isnan().all()             # without a list
    assert (cache.attend(q, pos, table, blocks=torch.full_like(blocks, -1)) == 0).all()
    assert (cache.attend(q, torch.zeros_like(pos), table, blocks=blocks.where(blocks > 0, -1)) == 0).all()
    # a window of which the list names no position: page 0 alone, far behind
    first = torch.zeros_like(blocks[..., :1])
    assert (cache.attend(q, pos, table, blocks=first, window=5) == 0).all()
    # where one page is finite, the others weigh nothing
    cache.k[table[:, 1].long()] = held[table[:, 1].long()]
    some = cache.attend(q, pos, table, blocks=blocks)
    one = torch.full_like(blocks, -1)
    one[..., 0] = 1
    alone = cache.attend(q, pos, table, blocks=one)
    assert torch.isfinite(some).all()
    # two roundings of an output, and twice 2^-14 of it (oracle.paged.attend_tolerance)
    assert (some.float() - alone.float()).abs().max() <= 2 * torch.finfo(dtype).eps * v.abs().max().item()


def test_scores_of_minus_infinity_by_a_negative_scale_and_in_part():
    g = gen(2)
    cache, table, k, v = filled(g, 1, 6, 16, 1, 64, BF16)
    q, pos = normal(g, 1, 1, 2, 64), torch.tensor([[60]], device=DEV)
    q[..., 3] = 2.0
    cache.k[..., 3] = INF
    blocks = torch.tensor([0, 3], dtype=torch.int32, device=DEV).view(1, 1, 1, 2)
    assert cache.attend(q, pos, table, blocks=blocks, scale=-0.125).isnan().all()
    q[:, :, 1, 3] = -2.0             # the other head of the group: +inf, a NaN by itself
    assert cache.attend(q, pos, table, blocks=blocks, scale=-0.125).isnan().all()
    q[:, :, 1, 3] = 0.0              # 0 times inf
    assert cache.attend(q, pos, table, blocks=blocks, scale=-0.125).isnan().all()

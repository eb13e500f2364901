"""Bounds behind a rotation: tokens past its tables store nothing, and leave
the bounds of their pages alone."""
import pytest
import torch

import epure
from epure.kernels import _abi, cuda
from test_gpu_bounds_shared import made
from test_gpu_select import BF16, DEV, E4M3, F16, I8, check_bounds, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def step(g, cache, table, pos, rotary):
    xdt = cache.dtype if cache.dtype.itemsize == 2 else BF16
    before = [cache.k.view(torch.uint8).clone(), cache.k_bounds.clone()]
    k, v, q = (normal(g, *pos.shape, cache.heads, cache.dim, dtype=xdt) for _ in range(3))
    cache.append(k, v, pos, table, q=q, rotary=rotary)
    check_bounds(cache, before[1], table.cpu(), pos.where(pos < rotary.max_pos, -1).cpu(), cache.page)
    return before


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("page,heads,D,limit,width", [(16, 2, 64, 90, 12), (32, 1, 128, 64, 4), (64, 8, 32, 1001, 130), (1024, 1, 16, 5, 1)])
def test_positions_on_both_sides_of_the_tables_end(page, heads, D, limit, width, dtype, native, monkeypatch):
    """Prompts in order and in none, one token, and tokens of which none is stored."""
    if not native:
        monkeypatch.setattr(_abi, "call", None)
    g = gen(limit)
    cache = made(g, 3 * width, page, heads, D, dtype)
    rotary = epure.Rotary(D, limit, device=DEV)
    table = torch.randperm(3 * width, generator=g, device=DEV).to(torch.int32).view(3, width)
    L = width * page
    n = min(L, 2 * limit)
    pos = torch.arange(n, device=DEV).repeat(3, 1)
    pos[1] += limit - 3
    pos[2] = pos[2, torch.randperm(n, generator=g, device=DEV)]
    step(g, cache, table, pos, rotary)
    for p in (limit - 1, limit, limit + 1, L - 1, 0):
        step(g, cache, table, torch.tensor([[p], [p - 1], [p + page]], device=DEV), rotary)
    held, limits = step(g, cache, table, limit + torch.arange(7, device=DEV).expand(3, 7), rotary)
    assert torch.equal(cache.k.view(torch.uint8), held) and torch.equal(cache.k_bounds, limits)


def test_sequences_of_one_page_on_both_sides():
    """The last token that is stored decides, not the last one."""
    g = gen(3)
    cache = made(g, 2, 64, 1, 32, BF16)
    rotary = epure.Rotary(32, 40, device=DEV)
    table = torch.zeros(5, 2, dtype=torch.int32, device=DEV)
    table[:, 1] = 1
    for S in (1, 3):
        step(g, cache, table, torch.tensor([[30], [39], [40], [5], [63]], device=DEV) - torch.arange(S, device=DEV), rotary)

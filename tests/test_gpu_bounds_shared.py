"""Bounds of pages that several sequences of one call write: rows up to the
largest position of all of the call's tokens on a page, whichever sequence it
belongs to."""
import pytest
import torch

import epure
from epure.kernels import cuda
from test_gpu_select import BF16, DEV, E4M3, F16, I8, check_bounds, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def made(g, pages, page, heads, D, dtype):
    """A cache of rows that some earlier use left, far wider than what the tests store."""
    cache = epure.PagedKVCache(pages, page, heads, D, dtype, DEV, bounds=True)
    k = normal(g, 1, pages * page, heads, D, dtype=dtype if dtype.itemsize == 2 else BF16, std=100.0)
    cache.append(k, k, torch.arange(pages * page, device=DEV), torch.arange(pages, device=DEV, dtype=torch.int32)[None])
    return cache


def step(g, cache, table, pos):
    xdt = cache.dtype if cache.dtype.itemsize == 2 else BF16
    before = cache.k_bounds.clone()
    k, v = (normal(g, *pos.shape, cache.heads, cache.dim, dtype=xdt) for _ in range(2))
    cache.append(k, v, pos, table)
    check_bounds(cache, before, table.cpu(), pos.cpu(), cache.page)


CHUNKS = [  # B, S, page, heads, D
    (2, 8, 16, 1, 32), (3, 24, 16, 2, 64), (5, 40, 32, 3, 80), (70, 3, 16, 2, 128), (9, 500, 16, 8, 16), (2, 700, 64, 1, 256),
    (4, 1030, 1024, 2, 48)]


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,page,heads,D", CHUNKS)
def test_a_prompt_in_chunks_over_one_table(B, S, page, heads, D, dtype):
    """Chunks in order, backwards, of tokens in no order, and dealt out one by one, each ending within a page."""
    g = gen(B * S)
    width = -(-B * S // page) + 1
    cache = made(g, width + 2, page, heads, D, dtype)
    table = torch.randperm(width + 2, generator=g, device=DEV)[:width].to(torch.int32)[None].expand(B, -1)
    pos = torch.arange(B * S, device=DEV).view(B, S)
    mixed = pos.flatten()[torch.randperm(B * S, generator=g, device=DEV)].view(B, S)
    for p in (pos, pos.flip(0), pos.flip(1), mixed, torch.where(pos % 7 == 3, -1, pos), pos.view(S, B).T,
              torch.where(torch.arange(B, device=DEV)[:, None] % 2 == 1, pos - 5, pos).clamp(min=0)):
        step(g, cache, table, p)


@pytest.mark.parametrize("dtype", [BF16, I8])
@pytest.mark.parametrize("B,page,heads,D", [(2, 16, 1, 16), (16, 16, 2, 128), (64, 64, 8, 128), (300, 1024, 1, 64), (129, 32, 3, 256)])
def test_one_token_each_on_common_pages(B, page, heads, D, dtype):
    g = gen(B)
    width = -(-B // page) + 2
    cache = made(g, width + 1, page, heads, D, dtype)
    table = torch.randperm(width + 1, generator=g, device=DEV)[:width].to(torch.int32)[None].expand(B, -1).contiguous()
    pos = torch.arange(B, device=DEV)[:, None]
    for p in (pos, pos.flip(0), pos + page - 1, torch.where(pos % 3 == 1, -1, pos), torch.full_like(pos, page + 3),
              torch.randint(-1, width * page + 2, (B, 1), generator=g, device=DEV)):
        step(g, cache, table, p)


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,heads", [(2100, 1, 5), (4200, 1, 3), (1100, 3, 8), (830, 17, 12)])
def test_more_sequences_than_workgroups_at_once(B, S, heads, dtype):
    """A workgroup takes two heads or three; every fifth sequence has the page of the one before."""
    assert B * heads >= 8192
    g = gen(B)
    cache = made(g, B + 3, 32, heads, 16, dtype)
    table = torch.randperm(B + 3, generator=g, device=DEV)[:B].to(torch.int32)[:, None].contiguous()
    table[4::5] = table[3::5][:table[4::5].shape[0]]
    start = torch.randint(-2, 32 - S + 1, (B, 1), generator=g, device=DEV)
    step(g, cache, table, start + torch.arange(S, device=DEV))
    step(g, cache, table, torch.where(start >= 0, start + torch.arange(S, device=DEV).flip(0), -1))


@pytest.mark.parametrize("S", [1, 5, 90])
def test_sequences_that_part_within_their_tables(S):
    """The first pages in common, the rest their own (or none, or nonsense): tokens on both."""
    g = gen(S)
    B, shared, own, page = 75, 4, 3, 32
    cache = made(g, shared + 40 * own, page, 2, 64, BF16)
    table = torch.full((B, shared + own), -1, dtype=torch.int32, device=DEV)
    table[:, :shared] = torch.arange(shared, dtype=torch.int32, device=DEV)
    table[:40, shared:] = shared + torch.arange(40 * own, dtype=torch.int32, device=DEV).view(40, own)
    table[70] = 0
    table[70, 0] = 1 << 20
    for lo in (0, 64, 100, 120):
        start = torch.randint(lo, shared * page + 5, (B, 1), generator=g, device=DEV)
        pos = start + torch.arange(S, device=DEV)
        pos[70] = -1
        step(g, cache, table, pos)


def test_a_replayed_step_on_common_pages():
    g = gen(6)
    cache = made(g, 4, 64, 2, 64, BF16)
    twin = epure.PagedKVCache.of(*(None if t is None else t.clone() for t in cache._held()))
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV).expand(8, 2)
    k, v, pos = normal(g, 8, 1, 2, 64), normal(g, 8, 1, 2, 64), torch.arange(8, device=DEV)[:, None]
    cache.append(k, v, pos, table)
    twin.append(k, v, pos, table)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(k, v, pos, table)
    for _ in range(4):
        k.copy_(normal(g, *k.shape))
        pos.copy_(torch.randperm(128, generator=g, device=DEV)[:8, None])
        graph.replay()
        twin.append(k, v, pos, table)
        torch.cuda.synchronize()
        assert torch.equal(cache.k_bounds, twin.k_bounds)


@pytest.mark.parametrize("S", [1, 70])
def test_bounds_of_rows_that_are_there_already(S):
    """The entry point without an append, behind one into a cache that keeps none."""
    import ctypes

    from epure.kernels import _abi
    from epure.paged import _tokens
    g = gen(S)
    B, page = 6, 16
    cache = made(g, 40, page, 2, 80, F16)
    bare = epure.PagedKVCache.of(cache.k, cache.v)
    table = torch.arange(40, dtype=torch.int32, device=DEV)[None].expand(B, -1)
    pos = torch.arange(B * S, device=DEV).view(B, S) + 5
    k = normal(g, B, S, 2, 80, dtype=F16)
    bare.append(k, k, pos, table)
    before = cache.k_bounds.clone()
    tok, _keep = _tokens((B, S), pos, table)
    assert _abi.lib.ep_kv_bounds(ctypes.byref(tok), ctypes.byref(cache._cache()), cache.k_bounds.data_ptr(),
                                 _abi.stream_handle(DEV)) == 0
    check_bounds(cache, before, table.cpu(), pos.cpu(), page)

"""Bounds of a cache's pages, the pages selected by them and attention over
those, against the plain restatements of oracle/paged.py."""
import pytest
import torch

import epure
from epure.kernels import cuda
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
TYPES = [BF16, F16, I8, E4M3]


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=BF16, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def made(g, B, width, page, heads, D, dtype, spare=3):
    cache = epure.PagedKVCache(B * width + spare, page, heads, D, dtype, DEV, bounds=True)
    table = torch.randperm(B * width + spare, generator=g, device=DEV)[:B * width].to(torch.int32).view(B, width)
    return cache, table


def held(t, s):
    x = t.float()
    return (x if s is None else x * s[..., None]).cpu()


def check_bounds(cache, before, table, pos, page):
    """Pages that the call's tokens lie on: their rows up to the largest position; the others as they were."""
    want, keys = before.cpu().float().clone(), held(cache.k, cache.k_scale)
    last = {}
    for b in range(pos.shape[0]):
        for p in pos[b].tolist():
            if p >= 0 and p // page < table.shape[1] and 0 <= int(table[b, p // page]) < cache.n_pages:
                i = int(table[b, p // page])
                last[i] = max(last.get(i, 0), p % page)
    for i, r in last.items():
        for h in range(cache.heads):
            want[i, h] = op.bounds(keys[i, h, :r + 1])
    got = cache.k_bounds.cpu().float()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))


# ------------------------------------------------------------------ bounds
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,width,page,heads,D", [(1, 1, 16, 1, 16), (3, 5, 16, 2, 128), (2, 3, 64, 3, 80),
                                                  (5, 2, 32, 1, 256), (2, 1, 1024, 1, 48), (2, 9, 16, 1, 144)])
def test_bounds_of_prompts_then_tokens(B, width, page, heads, D, dtype):
    """Bit for bit: minimum and maximum round nothing, and the held values are codes times scales in float32."""
    g = gen(B * D)
    cache, table = made(g, B, width, page, heads, D, dtype)
    assert cache.k_bounds.dtype == (dtype if dtype.itemsize == 2 else F32)
    L = width * page
    n = torch.randint(0, L + 1, (B, 1), generator=g, device=DEV)
    n[0] = L
    pos = torch.arange(L, device=DEV).expand(B, L)
    pos = torch.where(pos < n, pos, -1)
    xdt = dtype if dtype.itemsize == 2 else BF16

    def step(pos):
        before = cache.k_bounds.clone()
        k, v = (normal(g, B, pos.shape[1], heads, D, dtype=xdt) for _ in range(2))
        cache.append(k, v, pos, table)
        check_bounds(cache, before, table.cpu(), pos.cpu(), page)
    step(pos)
    step(torch.randint(-1, L + 3, (B, 1), generator=g, device=DEV))       # one token, back in the middle of a page
    step(torch.stack([torch.randperm(L, generator=g, device=DEV)[:min(L, 9)] for _ in range(B)]))     # in any order
    step(torch.randperm(L, generator=g, device=DEV).expand(B, L))


@pytest.mark.parametrize("dtype,page,D", [(BF16, 16, 48), (I8, 32, 80), (F16, 16, 256), (E4M3, 64, 128)])
def test_bounds_of_rows_that_more_workgroups_share(dtype, page, D):
    """Rows of more than 64 groups of 64 tokens, past 1024 pages: one in order, one in order with gaps that ends
    early, one in order but for its last token, one that begins with none, one backwards."""
    S, B, heads = 4200, 5, 16 if page == 64 else 4
    g = gen(page)
    cache, table = made(g, B, -(-S // page) + 2, page, heads, D, dtype)
    pos = torch.arange(S, device=DEV).repeat(B, 1)
    pos[1] = (pos[1] + pos[1] // 5).where(pos[1] < 3000, -1)
    pos[2, -1] = 7
    pos[3] = torch.where(pos[3] < 70, -1, pos[3] - 70)
    pos[4] = pos[4].flip(0)
    xdt = dtype if dtype.itemsize == 2 else BF16
    for _ in range(2):
        before = cache.k_bounds.clone()
        cache.append(normal(g, B, S, heads, D, dtype=xdt), normal(g, B, S, heads, D, dtype=xdt), pos, table)
        check_bounds(cache, before, table.cpu(), pos.cpu(), page)
        pos = pos[:, torch.randperm(S, generator=g, device=DEV)]        # then in no order at all


def test_bounds_through_a_rotation_with_queries_and_without_the_native_path(monkeypatch):
    from epure.kernels import _abi
    g = gen(3)
    r = epure.Rotary(64, 90, device=DEV)
    k, v, q = normal(g, 2, 70, 2, 64), normal(g, 2, 70, 2, 64), normal(g, 2, 70, 4, 64)
    pos = torch.arange(70, device=DEV)
    got = []
    for native in (True, False):
        cache, table = made(gen(4), 2, 5, 16, 2, 64, BF16)
        if not native:
            monkeypatch.setattr(_abi, "call", None)
        before = cache.k_bounds.clone()
        cache.append(k, v, pos, table, q=q, rotary=r)
        check_bounds(cache, before, table.cpu(), pos.expand(2, 70).cpu(), 16)
        got.append(cache.k_bounds)
    assert torch.equal(*got)


def test_bounds_of_rows_that_are_not_finite_and_of_pages_that_are_not_there():
    g = gen(5)
    cache, table = made(g, 2, 4, 16, 1, 32, BF16)
    k, v = normal(g, 2, 64, 1, 32), normal(g, 2, 64, 1, 32)
    k[0, 3, 0, 5], k[0, 20, 0, 1], k[1, 40, 0, 2] = float("nan"), float("inf"), float("-inf")
    table[0, 3], table[1, 0] = -1, 1000
    before = cache.k_bounds.clone()
    cache.append(k, v, torch.arange(64, device=DEV), table)
    check_bounds(cache, before, table.cpu(), torch.arange(64).expand(2, 64), 16)
    assert cache.k_bounds.isnan().sum() == 2 and cache.k_bounds.isinf().sum() == 2


# ------------------------------------------------------------------ selection
def limits(cache, table):
    """Bounds of each sequence's pages in order, NaN where the pool has none."""
    t, b = table.cpu().long(), cache.k_bounds.cpu().float()
    ok = (t >= 0) & (t < cache.n_pages)
    return torch.where(ok[..., None, None, None], b[torch.where(ok, t, 0)], torch.nan)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,width,page,G,heads,D,take", [
    (1, 1, 1, 16, 1, 1, 16, 1), (3, 1, 9, 16, 4, 2, 128, 4), (2, 3, 40, 16, 3, 1, 96, 7), (2, 1, 5, 32, 8, 2, 256, 9),
    (1, 2, 300, 16, 1, 1, 48, 64), (2, 1, 700, 16, 3, 2, 80, 100), (2, 1, 150, 16, 5, 2, 80, 149), (1, 1, 33, 64, 2, 1, 144, 1), (4, 1, 7, 16, 2, 1, 64, 7)])
def test_selection(B, S, width, page, G, heads, D, take, dtype):
    """Equal pages: scores in float64 differ by far more than their sums' rounding."""
    g = gen(width + take)
    cache, table = made(g, B, width, page, heads, D, dtype)
    cache.k_bounds.copy_(normal(g, *cache.k_bounds.shape, dtype=F32).sort(2).values)
    q = normal(g, B, S, G * heads, D, dtype=F16 if dtype == F16 else BF16, std=2.0)
    L = width * page
    pos = torch.randint(0, L, (B, S), generator=g, device=DEV)
    pos.view(-1)[0] = L - 1
    pos.view(-1)[1:4] = torch.tensor([-1, L, 0], device=DEV)[:max(B * S - 1, 0)]
    got = cache.select(q, pos, table, take)
    assert got.dtype == torch.int32
    assert torch.equal(got.cpu(), op.select(q, limits(cache, table), pos, page, take))


def test_equal_scores_go_to_the_lower_page_and_nan_is_above_all():
    g = gen(7)
    cache, table = made(g, 1, 500, 16, 2, 32, BF16)
    q = torch.ones(1, 1, 2, 32, dtype=BF16, device=DEV)
    pos = torch.tensor([[499 * 16 + 3]], device=DEV)
    value = torch.randint(0, 5, (503, 2, 1, 1), generator=g, device=DEV).to(BF16)
    cache.k_bounds.copy_(value.expand(503, 2, 2, 32))
    for take in (1, 2, 50, 100, 101, 499, 500, 600):
        assert torch.equal(cache.select(q, pos, table, take).cpu(), op.select(q, limits(cache, table), pos, 16, take))
    cache.k_bounds[table[0, 40].long(), 0, 1, 3] = float("nan")
    cache.k_bounds[table[0, 41].long(), 1, 0, 3] = float("inf")
    table[0, 77] = -5
    cache.k_bounds.mul_(-1.0)
    for take in (2, 3, 4, 200):
        got = cache.select(q, pos, table, take).cpu()
        want = op.select(q, limits(cache, table), pos, 16, take)
        assert torch.equal(got, want)


def test_scores_that_float32_could_not_tell_apart():
    """Column 0 is large and alike, column 1 parts the pages below its float32 step."""
    cache, table = made(gen(8), 1, 64, 16, 1, 32, I8)
    cache.k_bounds.zero_()
    cache.k_bounds[..., 0] = 3.0e6
    order = torch.randperm(64, generator=gen(9), device=DEV)
    cache.k_bounds[table[0].long(), 0, :, 1] = (order * 2.0 ** -12)[:, None].float()
    q = torch.ones(1, 1, 1, 32, dtype=BF16, device=DEV)
    got = cache.select(q, torch.tensor([[63 * 16]], device=DEV), table, 9)[0, 0, 0]
    want = order[:63].argsort(descending=True)[:8].sort().values
    assert torch.equal(got[:8].long(), want) and got[8] == 63


def test_more_pages_than_are_held_in_lds():
    g = gen(10)
    B, width, page = 2, 9000, 16
    cache = epure.PagedKVCache(64, page, 1, 16, BF16, DEV, bounds=True)
    cache.k_bounds.copy_(normal(g, 64, 1, 2, 16))
    table = torch.randint(0, 64, (B, width), generator=g, device=DEV).to(torch.int32)     # many equal scores
    q = normal(g, B, 1, 2, 16)
    pos = torch.tensor([[width * page - 1], [4097 * page]], device=DEV)
    for take in (2, 100, 5000):
        got = cache.select(q, pos, table, take)
        assert torch.equal(got.cpu(), op.select(q, limits(cache, table), pos, page, take))


# ------------------------------------------------------------------ attention over a list
def filled(g, B, width, page, heads, D, dtype):
    cache, table = made(g, B, width, page, heads, D, dtype)
    xdt = dtype if dtype.itemsize == 2 else BF16
    L = width * page
    k, v = normal(g, B, L, heads, D, dtype=xdt), normal(g, B, L, heads, D, dtype=xdt)
    cache.append(k, v, torch.arange(L, device=DEV), table)
    return cache, table, op.stands_for(k, dtype), op.stands_for(v, dtype)


def check(got, q, k, v, pos, blocks, page, scale, window=None):
    out, mag, big = op.attend_blocks(q, k, v, pos, blocks, page, scale, window)
    assert torch.equal(got.cpu().isnan(), out.isnan())
    ok = ~out.isnan()
    tol = op.attend_tolerance(out, mag, big, got.dtype, q.shape[-1])
    bad = (got.cpu().double() - out).abs()[ok] > tol[ok]
    assert not bad.any(), f"{bad.sum().item()} of {bad.numel()} off"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,S,width,page,G,heads,D,take", [
    (1, 1, 1, 16, 1, 1, 16, 1), (3, 1, 9, 16, 4, 2, 128, 4), (2, 3, 20, 16, 3, 1, 96, 7), (2, 1, 5, 32, 8, 2, 256, 9),
    (1, 2, 30, 16, 17, 1, 48, 21), (2, 1, 40, 16, 5, 2, 80, 39), (1, 1, 33, 64, 2, 1, 144, 32), (2, 1, 7, 128, 40, 1, 192, 3),
    (5, 2, 6, 16, 1, 2, 160, 5), (1, 1, 3, 1024, 2, 1, 112, 2)])
def test_attention_over_a_list(B, S, width, page, G, heads, D, take, dtype):
    """Pages in any order, behind the token, unnamed, past the table; windows; rows without a page."""
    g = gen(width + D)
    cache, table, k, v = filled(g, B, width, page, heads, D, dtype)
    q = normal(g, B, S, G * heads, D, dtype=dtype if dtype.itemsize == 2 else F16 if D % 48 == 0 else BF16, std=2.0)
    L = width * page
    pos = torch.randint(0, L, (B, S), generator=g, device=DEV)
    pos.view(-1)[0] = L - 1
    pos.view(-1)[1:3] = torch.tensor([-1, L], device=DEV)[:max(B * S - 1, 0)]
    blocks = torch.rand(B, S, heads, max(width, take), generator=g, device=DEV).argsort(-1)[..., :take].to(torch.int32)
    lists = [blocks, torch.where(torch.rand(blocks.shape, generator=g, device=DEV) < 0.4, -1, blocks),
             torch.full_like(blocks, -1), blocks + (1 << 30), cache.select(q, pos, table, take)]
    for x in lists:
        check(cache.attend(q, pos, table, blocks=x), q, k, v, pos, x, page, D ** -0.5)
    check(cache.attend(q, pos, table, blocks=blocks, window=page + 5, scale=0.2), q, k, v, pos, blocks, page, 0.2, page + 5)
    every = torch.arange(width, device=DEV, dtype=torch.int32).expand(B, S, heads, width)
    out, mag, big = op.attend(q, k, v, pos, D ** -0.5)
    got = cache.attend(q, pos, table, blocks=every).cpu().double()
    assert torch.equal(got.isnan(), out.isnan())
    assert ((got - out).abs() <= op.attend_tolerance(out, mag, big, q.dtype, D))[~out.isnan()].all()


def test_a_page_named_twice_counts_twice():
    g = gen(11)
    cache, table, k, v = filled(g, 1, 4, 16, 1, 64, BF16)
    q, pos = normal(g, 1, 1, 2, 64), torch.tensor([[60]], device=DEV)
    blocks = torch.tensor([2, 0, 2, 2], dtype=torch.int32, device=DEV).view(1, 1, 1, 4)
    check(cache.attend(q, pos, table, blocks=blocks), q, k, v, pos, blocks, 16, 0.125)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_missing_pages_and_values_that_are_not_finite(dtype):
    """On a page that is not listed, or behind the token, they reach nobody."""
    g = gen(12)
    cache, table, k, v = filled(g, 1, 6, 16, 1, 64, dtype)
    q, pos = normal(g, 1, 1, 2, 64, std=2.0), torch.tensor([[68]], device=DEV)
    table = table.clone()
    cache.k[int(table[0, 1])] = float("nan")                          # page 1
    cache.v[int(table[0, 4]), 0, 5:] = float("nan")                  # rows behind position 68
    table[0, 2] = -1
    for pages, bad in (([0, 3, 4, -1], False), ([4, -1, 5, -1], False), ([0, 1, 4, -1], True), ([2, 0, 3, 4], True)):
        got = cache.attend(q, pos, table, blocks=torch.tensor(pages, dtype=torch.int32, device=DEV).view(1, 1, 1, 4))
        assert got.isnan().all() == bad and got.isnan().any() == bad


def test_a_step_of_all_three_replays_in_a_graph():
    """append with bounds, select, attend: each replay as the eager calls, with eager work between."""
    g = gen(13)
    cache, table, *_ = filled(g, 3, 30, 16, 2, 64, I8)
    twin = epure.PagedKVCache.of(*(t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale, cache.k_bounds)))
    k, v, q = (normal(g, 3, 1, h, 64) for h in (2, 2, 6))
    pos = torch.tensor([[470], [3], [200]], device=DEV)

    def step(c):
        c.append(k, v, pos, table)
        blocks = c.select(q, pos, table, 5)
        return blocks, c.attend(q, pos, table, blocks=blocks)
    step(twin)
    step(cache)         # the same history in both
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for i in range(4):
        for t in (k, v, q):
            t.copy_(normal(g, *t.shape))
        pos.copy_(torch.randint(-1, 480, (3, 1), generator=g, device=DEV))
        graph.replay()
        want = step(twin)
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        assert torch.equal(cache.k_bounds, twin.k_bounds)


def test_native_and_python_paths_are_the_same(monkeypatch):
    from epure.kernels import _abi
    g = gen(14)
    cache, table, *_ = filled(g, 2, 12, 16, 2, 96, F16)
    q, pos = normal(g, 2, 2, 4, 96, dtype=F16), torch.randint(0, 192, (2, 2), generator=g, device=DEV)
    wide = torch.stack((q, q), 3).flatten(2, 3)[:, :, ::2]

    def calls():
        b = cache.select(q, pos, table, 4)
        return b, cache.select(wide, pos, table, 20), cache.attend(q, pos, table, blocks=b), \
            cache.attend(wide, pos[:, :1], table, blocks=b, window=50), \
            cache.attend(q, pos, table, blocks=torch.cat((b, b), -1)[..., ::2]), cache.attend(q, pos, table[:, ::2], shared=2)
    native = calls()
    monkeypatch.setattr(_abi, "call", None)
    for a, b in zip(native, calls()):
        assert torch.equal(a.float().nan_to_num(7.0), b.float().nan_to_num(7.0))


def test_refusals():
    g = gen(15)
    cache, table, *_ = filled(g, 2, 3, 16, 1, 64, BF16)
    bare = epure.PagedKVCache.of(cache.k, cache.v)
    q, pos = normal(g, 2, 1, 2, 64), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    b = torch.zeros(2, 1, 1, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="bounds"):
        bare.select(q, pos, table, 2)
    for bad, error in (((q, pos, table, 0), ValueError), ((q, pos, table, 1.5), TypeError), ((q.float(), pos, table, 2), TypeError),
                       ((q[..., :48], pos, table, 2), ValueError), ((q, pos, table.long(), 2), TypeError),
                       ((q, pos.float(), table, 2), TypeError), ((q[:, :, :0], pos, table, 2), ValueError),
                       ((q, pos, table, 1 << 27), ValueError)):
        with pytest.raises(error):
            cache.select(*bad)
    for bad, error in ((b.long(), TypeError), (b[:1], ValueError), (b[..., :0], ValueError), (b[0], ValueError),
                       (b.expand(2, 1, 2, 2), ValueError), (b.cpu(), ValueError)):
        with pytest.raises(error):
            cache.attend(q, pos, table, blocks=bad)
    with pytest.raises(RuntimeError, match="no backward"):
        cache.select(q.clone().requires_grad_(), pos, table, 2)
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(cache.k, cache.v, k_bounds=cache.k_bounds[:2])
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(cache.k, cache.v, k_bounds=cache.k_bounds.float())
    assert cache.select(q[:0], pos[:0], table[:0], 2).shape == (0, 1, 1, 2)

"""Attention behind shared pages with so many rows that those pages go through
LDS (csrc/attend_front.h), against a softmax over each row's positions in
float64 on the GPU."""
import math

import pytest
import torch

import epure
from epure.kernels import cuda
from oracle import paged as op
from test_gpu_shared import BF16, DEV, E4M3, F16, I8, gen, normal, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def filled(g, B, shared, own, page, heads, D, dtype):
    """A cache and what it holds: shared [P, heads, D] and own [B, L, heads, D], keys and values, float64 on the GPU."""
    cache = epure.PagedKVCache(shared + B * own + 2, page, heads, D, dtype, DEV)
    table = tables(g, B, shared, own)
    xdt = dtype if dtype.itemsize == 2 else BF16
    P, L = shared * page, own * page
    parts = []
    for n, rows, at, tab in ((1, P, 0, table[:1, :shared]), (B, L, P, table)):
        k, v = (normal(g, n, rows, heads, D, dtype=xdt) for _ in range(2))
        pos = (at + torch.arange(rows, device=DEV)).expand(n, rows)
        cache.append(k, v, pos, tab)
        parts.append([x.double() for x in cache.read(pos, tab, torch.float32)])      # codes times scales
    return cache, table, parts


def reference(q, parts, pos, scale, window=None):
    """(output, sum of weight * |v|, largest sum of |q k| times scale), as oracle.paged.attend."""
    B, S, H, D = q.shape
    (ks, vs), (ko, vo) = parts
    P, L, heads = ks.shape[1], ko.shape[1], ks.shape[2]
    G = H // heads
    q = q.double().view(B, S, heads, G, D)
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    big = torch.zeros(B, S, heads, G, 1, dtype=torch.float64, device=DEV)
    j = torch.arange(P + L, device=DEV)
    for b in range(B):
        p = pos[b][:, None]
        see = (j <= p) & (p >= 0)
        if window:
            see &= j > p - window
        lo, hi = int(see.any(0).int().argmax()), P + L        # a plain form too may leave out what no row sees
        k, v = (torch.cat((x[0], y[b]))[lo:hi].transpose(0, 1).contiguous() for x, y in ((ks, ko), (vs, vo)))
        x = q[b].transpose(0, 1).reshape(heads, S * G, D)
        ok = see[:, None, lo:hi].expand(S, G, -1).reshape(S * G, -1)
        back = lambda t: t.view(heads, S, G, -1).transpose(0, 1)  # noqa: E731
        kt = k.transpose(1, 2).contiguous()
        w = torch.softmax((x @ kt * scale).masked_fill(~ok, -math.inf), -1).nan_to_num(0.0)
        out[b], mag[b] = back(w @ v), back(w @ v.abs())
        big[b] = back((x.abs() @ kt.abs() * abs(scale)).masked_fill(~ok, 0.0).amax(-1))
    out = torch.where((pos >= P + L)[:, :, None, None, None], torch.nan, out)
    return [t.reshape(B, S, H, -1) for t in (out, mag, big)]


def check(got, want):
    out, mag, big = want
    assert torch.equal(got.isnan(), out.isnan())
    ok = ~out.isnan()
    tol = op.attend_tolerance(out, mag, big, got.dtype, got.shape[-1])
    bad = (got.double() - out).abs()[ok] > tol[ok]
    assert not bad.any(), f"{bad.sum().item()} of {bad.numel()} off"


def tiles(B, S, shared, page, G, heads, window=None):
    """Of 32 rows by 32 positions: from 16384 on the shared pages always go through LDS."""
    return -(-B * S * G // 32) * heads * (min(shared * page, window or shared * page) // 32)


CASES = [  # B, S, shared, own, page, G, heads, D
    (64, 1, 128, 2, 32, 8, 8, 128), (43, 3, 331, 2, 16, 2, 16, 64), (128, 1, 33, 1, 64, 8, 8, 96), (9, 5, 67, 1, 128, 5, 8, 80),
    (11, 1, 2, 1, 1024, 12, 64, 16), (33, 1, 1030, 1, 16, 1, 16, 48), (20, 8, 9, 1, 256, 3, 16, 112)]


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,shared,own,page,G,heads,D", CASES)
def test_many_rows(B, S, shared, own, page, G, heads, D, dtype):
    """Tokens behind the prefix; some inside it, at its ends, padded and past the table; windows over its end."""
    assert tiles(B, S, shared, page, G, heads) >= 16384
    g = gen(B * D + S)
    cache, table, parts = filled(g, B, shared, own, page, heads, D, dtype)
    q = normal(g, B, S, G * heads, D, dtype=dtype if dtype.itemsize == 2 else F16 if D % 48 == 0 else BF16, std=2.0)
    P, L = shared * page, (shared + own) * page
    pos = torch.randint(P, L, (B, S), generator=g, device=DEV)
    check(cache.attend(q, pos, table, shared=shared), reference(q, parts, pos, D ** -0.5))
    pos.view(-1)[:7] = torch.tensor([P - 1, P, L - 1, 0, -1, L, P // 2], device=DEV)
    check(cache.attend(q, pos, table, shared=shared, scale=-0.21), reference(q, parts, pos, -0.21))
    for window in (P - 33, P + 3):
        if tiles(B, S, shared, page, G, heads, window) >= 16384:
            check(cache.attend(q, pos, table, shared=shared, window=window), reference(q, parts, pos, D ** -0.5, window))


def three_ways(B, S, shared, own, page, G, heads, D, dtype):
    g = gen(B * D + S)
    cache, table, parts = filled(g, B, shared, own, page, heads, D, dtype)
    q = normal(g, B, S, G * heads, D, dtype=dtype if dtype.itemsize == 2 else F16 if D % 48 == 0 else BF16, std=2.0)
    P, L = shared * page, (shared + own) * page
    pos = torch.randint(P, L, (B, S), generator=g, device=DEV)
    check(cache.attend(q, pos, table, shared=shared), reference(q, parts, pos, D ** -0.5))
    pos.view(-1)[:7] = torch.tensor([P - 1, P, L - 1, 0, -1, L, P // 2], device=DEV)[:B * S]
    check(cache.attend(q, pos, table, shared=shared, scale=-0.21), reference(q, parts, pos, -0.21))
    check(cache.attend(q, pos, table, shared=shared, window=P - 3), reference(q, parts, pos, D ** -0.5, P - 3))


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,shared,own,page,G,heads,D", [
    (8, 5, 130, 1, 64, 8, 8, 128), (3, 33, 200, 2, 32, 3, 32, 64), (4, 12, 90, 1, 64, 4, 16, 96), (2, 70, 600, 5, 16, 1, 12, 48),
    (2, 70, 500, 5, 16, 1, 12, 48)])
def test_many_rows_of_each_sequence(B, S, shared, own, page, G, heads, D, dtype):
    """More than 32 on a cache head: the sequences' own pages in a launch of their own (the last case: no LDS)."""
    assert S * G > 32 and (tiles(B, S, shared, page, G, heads) >= 16384) == (shared != 500)
    three_ways(B, S, shared, own, page, G, heads, D, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("B,S,shared,own,page,G,heads,D", [
    (33, 1, 65, 1, 16, 1, 1, 64), (17, 1, 17, 40, 64, 2, 3, 128), (7, 1, 2, 1, 1024, 5, 2, 96), (4, 4, 9, 3, 128, 8, 2, 112),
    (2, 1, 33, 90, 32, 17, 1, 16), (40, 1, 33, 300, 32, 4, 8, 128), (300, 1, 17, 1, 64, 1, 2, 80), (9, 2, 80, 2, 16, 16, 1, 128)])
def test_few_tiles_and_long_contexts_behind_them(B, S, shared, own, page, G, heads, D, dtype):
    """33 rows on and few positions in common; own pages in one piece a sequence, or cut into shares."""
    assert B * S * G > 32 >= S * G and tiles(B, S, shared, page, G, heads) < 16384
    three_ways(B, S, shared, own, page, G, heads, D, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
def test_missing_pages_and_values_that_are_not_finite(dtype):
    """They reach who sees them, and nobody else."""
    B, S, shared, own, page, G, heads, D = 64, 1, 300, 2, 16, 4, 16, 64
    g = gen(5)
    cache, table, parts = filled(g, B, shared, own, page, heads, D, dtype)
    q = normal(g, B, S, G * heads, D, dtype=dtype if dtype.itemsize == 2 else BF16)
    pos = (4700 + 2 * torch.arange(B, device=DEV))[:, None]          # 4700 .. 4826, the prefix ends at 4800
    want = reference(q, parts, pos, 0.125)
    page_of = lambda p: int(table[0, p // page])  # noqa: E731
    if dtype.itemsize == 2:
        cache.v[page_of(4750), 3, 4750 % page, 9] = float("inf")
        cache.k[page_of(4763), 3, 4763 % page, 1] = float("nan")
    elif dtype == E4M3:
        cache.v.view(torch.uint8)[page_of(4750), 3, 4750 % page, 9] = 0x7f         # NaN
        cache.k_scale[page_of(4763), 3, 4763 % page] = float("nan")
    else:
        cache.v_scale[page_of(4750), 3, 4750 % page] = float("inf")
        cache.k_scale[page_of(4763), 3, 4763 % page] = float("nan")
    got = cache.attend(q, pos, table, shared=shared)
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[pos[:, 0] >= 4750, :, 3 * G:4 * G, slice(None) if dtype == I8 else slice(9, 10)] = True
    hit[pos[:, 0] >= 4763, :, 3 * G:4 * G] = True
    assert torch.equal(~got.isfinite(), hit)
    tol = op.attend_tolerance(*want, got.dtype, D)
    assert ((got.double() - want[0]).abs() <= tol)[~hit].all()
    table = table.clone()
    table[0, 4768 // page] = 1 << 20                 # positions 4768 .. 4783
    lost = cache.attend(q, pos, table, shared=shared)
    hit |= (pos >= 4768)[:, :, None, None]
    assert torch.equal(~lost.isfinite(), hit)
    assert torch.equal(lost[~hit], got[~hit])


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scores_that_grow_and_shrink_along_the_prefix(dtype):
    """Maxima that rise by little, by much and past 2^24, then long tails of small weights."""
    B, shared, page, G, heads, D = 64, 32, 64, 8, 16, 32
    g = gen(6)
    cache, table, parts = filled(g, B, shared, 1, page, heads, D, dtype)
    q = normal(g, B, 1, G * heads, D, dtype=dtype, std=0.5)
    q[..., 0] = 16.0
    P = shared * page
    ramp = torch.arange(P, device=DEV)
    for make in (lambda: ramp / 256.0, lambda: (P - ramp) / 128.0, lambda: (ramp % 640) / 8.0 - 40.0,
                 lambda: torch.where(ramp % 512 == 300, 3.0e4, -3.0e4)):
        k = parts[0][0].to(dtype)
        k[0, :, :, 0] = make()[:, None].to(dtype)
        cache.append(k, parts[0][1].to(dtype), ramp, table[:1])
        held = [[k.double(), parts[0][1]], parts[1]]
        pos = torch.randint(P, P + page, (B, 1), generator=g, device=DEV)
        for scale in (1.0, 64.0):
            check(cache.attend(q, pos, table, shared=shared, scale=scale), reference(q, held, pos, scale))


def test_graphs_and_streams():
    g = gen(7)
    B, shared, page, G, heads, D = 64, 64, 64, 4, 16, 64
    cache, table, parts = filled(g, B, shared, 1, page, heads, D, BF16)
    q = normal(g, B, 1, G * heads, D, std=2.0)
    pos = torch.randint(0, 65 * page, (B, 1), generator=g, device=DEV)
    want = cache.attend(q, pos, table, shared=shared)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.attend(q, pos, table, shared=shared)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.attend(q, pos, table, shared=shared)
    for _ in range(3):
        pos.copy_(torch.randint(0, 65 * page, (B, 1), generator=g, device=DEV))
        q.copy_(normal(g, *q.shape, std=2.0))
        want = cache.attend(q, pos, table, shared=shared)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)

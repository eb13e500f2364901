"""Attention over the paged cache where its work is shared among workers:
more units than one count takes, shares that begin and end inside segments,
contexts around the size at which sharing begins, and calls of many rows."""
import pytest
import torch

import epure
from epure.kernels import _abi, cuda
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


def filled(g, lengths, page, heads, dim, dtype, width=None):
    """A cache of random contexts on shuffled pages (unused ones hold NaN),
    its table, and what it holds [B, L, heads, D]."""
    rows = [-(-n // page) for n in lengths]
    n = sum(rows) + 2
    cache = epure.PagedKVCache(n, page, heads, dim, dtype, DEV)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(0xff if dtype.itemsize == 2 else 0x7f)
    for s in (cache.k_scale, cache.v_scale):
        if s is not None:
            s.fill_(float("nan"))
    order = torch.randperm(n, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lengths), width or max(max(rows), 1)), -7, dtype=torch.int32, device=DEV)
    at = 0
    for b, r in enumerate(rows):
        table[b, :r] = order[at:at + r]
        at += r
    top = max(max(lengths), 1)
    pos = torch.arange(top, device=DEV).expand(len(lengths), top).clone()
    for b, m in enumerate(lengths):
        pos[b, m:] = -1
    k, v = (normal(g, len(lengths), top, heads, dim, dtype=F32) for _ in range(2))
    cache.append(k, v, pos, table)
    return cache, table, op.stands_for(k, dtype), op.stands_for(v, dtype)


def check(cache, table, q, pos, kc, vc, rows=None, **kw):
    """Against the oracle, for the listed sequences (default: all)."""
    out = cache.attend(q, pos, table, **kw)
    rows = list(range(q.shape[0])) if rows is None else rows
    want, mag, big = op.attend(q[rows], kc[rows], vc[rows], pos[rows].cpu(), kw.get("scale", cache.dim ** -0.5),
                               kw.get("window"))
    tol = op.attend_tolerance(want, mag, big, q.dtype, cache.dim)
    err = (out[rows].cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-300)).max().item():.3g} of the tolerance"
    return out


@pytest.mark.parametrize("dtype", [BF16, I8])
def test_more_units_than_one_count_takes(dtype):
    """A wave counts the tiles of 64 sequences at a time."""
    g = gen(1)
    lengths = [(37 * i) % 900 for i in range(150)]
    lengths[0], lengths[64], lengths[149] = 1100, 0, 1500
    cache, table, kc, vc = filled(g, lengths, 32, 1, 64, dtype)
    q = normal(g, 150, 1, 3, 64, std=2.0)
    pos = torch.tensor(lengths, device=DEV)[:, None] - 1
    out = check(cache, table, q, pos, kc, vc)
    # each sequence alone gives the same up to the joins' rounding
    for b in (0, 63, 64, 65, 128, 149):
        one = cache.attend(q[b:b + 1], pos[b:b + 1], table[b:b + 1])
        assert torch.allclose(one.float(), out[b:b + 1].float(), rtol=2.0 ** -7, atol=1e-6)


@pytest.mark.parametrize("tiles", [1, 15, 16, 17, 31, 32, 33, 47])
@pytest.mark.parametrize("B,heads", [(2, 1), (33, 8)])
def test_contexts_around_the_size_at_which_sharing_begins(tiles, B, heads):
    g = gen(tiles)
    lengths = [max(32 * tiles - i, 0) for i in range(B)]
    cache, table, kc, vc = filled(g, lengths, 32, heads, 64, BF16, width=tiles)
    q = normal(g, B, 1, heads, 64, std=2.0)
    pos = torch.tensor(lengths, device=DEV)[:, None] - 1
    check(cache, table, q, pos, kc, vc, rows=[0, 1, B - 1])


@pytest.mark.parametrize("dtype,qdt", [(BF16, BF16), (F16, F16), (I8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_many_rows_over_long_contexts(D, dtype, qdt):
    """Rows of one and two tiles, and of several units, shared and joined;
    tokens of one call at different places."""
    g = gen(D)
    lengths = [1300, 5, 700]
    cache, table, kc, vc = filled(g, lengths, 64, 2, D, dtype)
    for S, G in ((3, 5), (4, 8), (9, 4)):
        q = normal(g, 3, S, 2 * G, D, dtype=qdt, std=2.0)
        pos = torch.tensor(lengths, device=DEV)[:, None] - S + torch.arange(S, device=DEV)
        pos[0, 0] = 17
        check(cache, table, q, pos, kc, vc)
        check(cache, table, q, pos, kc, vc, window=333)


def test_long_tail_of_small_weights_in_f16():
    """One large score and 30000 of 2^-17 of it: the tail is a fifth of the
    weight, each part of it below f16's least number relative to the largest."""
    n, D = 30000, 64
    cache = epure.PagedKVCache(n // 64 + 1, 64, 1, D, F16, DEV)
    table = torch.arange(n // 64 + 1, dtype=torch.int32, device=DEV)[None]
    pos = torch.arange(n, device=DEV)[None]
    k, v = torch.zeros(1, n, 1, D, device=DEV), torch.ones(1, n, 1, D, device=DEV)
    k[0, 777, 0, 0], v[0, 777] = 1.0, -1.0
    cache.append(k, v, pos, table)
    q = torch.zeros(1, 1, 1, D, dtype=F16, device=DEV)
    q[..., 0] = 12.0                                    # e^12 = 2^17.3
    check(cache, table, q, torch.tensor([[n - 1]], device=DEV), op.stands_for(k, F16), op.stands_for(v, F16),
          scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, E4M3])
def test_bad_pages_in_the_middle_give_nan_to_the_rows_that_need_them(dtype):
    g = gen(5)
    lengths = [1000, 1000]
    cache, table, kc, vc = filled(g, lengths, 16, 2, 64, dtype)
    pos = torch.tensor([[999, 400, 100], [999, 400, 100]], device=DEV)
    q = normal(g, 2, 3, 4, 64)
    bad = table.clone()
    bad[0, 20], bad[1, 62] = cache.n_pages, -1          # positions 320 .. 335; 992 .. 1007
    for window in (None, 150):
        want = cache.attend(q, pos, table, window=window)
        out = cache.attend(q, pos, bad, window=window)
        hit = torch.tensor([[window is None, True, False], [True, False, False]])
        assert torch.equal(out.isnan().all(-1).all(-1).cpu(), hit)
        assert torch.equal(out[~hit.to(DEV)], want[~hit.to(DEV)])


def test_infinite_scores():
    """A key of -inf in the scores weighs nothing; +inf, or nothing but -inf, is NaN."""
    cache = epure.PagedKVCache(40, 16, 1, 64, BF16, DEV)
    table = torch.arange(40, dtype=torch.int32, device=DEV)[None]
    g = gen(6)
    k, v = normal(g, 1, 600, 1, 64, dtype=F32), normal(g, 1, 600, 1, 64, dtype=F32)
    q = torch.ones(1, 3, 1, 64, dtype=BF16, device=DEV)
    k[0, 0], k[0, 300, 0, 5], k[0, 590, 0, 6] = -torch.inf, -torch.inf, torch.inf
    pos = torch.arange(600, device=DEV)[None]
    cache.append(k, v, pos, table)
    kc, vc = op.stands_for(k, BF16), op.stands_for(v, BF16)
    rows = torch.tensor([[0, 580, 599]], device=DEV)
    out = cache.attend(q, rows, table)
    assert out[0, 0].isnan().all() and out[0, 2].isnan().all() and torch.isfinite(out[0, 1]).all()
    kc[0, 0], kc[0, 300] = -1e4, -1e4                   # as good as -inf, and finite for the oracle
    want, mag, _ = op.attend(q[:, 1:2], kc, vc, rows[:, 1:2].cpu(), 0.125)
    big = (kc[0, 1:581, 0].abs().sum(-1) * 0.125)[torch.arange(580) != 299].max()
    tol = op.attend_tolerance(want, mag, big, BF16, 64)
    assert ((out[:, 1:2].cpu().double() - want).abs() <= tol).all()


def test_a_workspace_that_is_too_small_is_refused():
    cache = epure.PagedKVCache(64, 16, 1, 64, BF16, DEV)
    table = torch.zeros(1, 64, dtype=torch.int32, device=DEV)
    q, pos = normal(gen(7), 1, 1, 4, 64), torch.zeros(1, 1, dtype=torch.int64, device=DEV)
    heads = _abi.Heads(q.data_ptr(), _abi.BF16, 4, 256, 256, 64)
    tok = _abi.Tokens(1, 1, pos.data_ptr(), 1, 1, table.data_ptr(), 64, 64)
    need = _abi.lib.ep_paged_attention_workspace(heads, tok, cache._cache())
    assert need > 0
    ws, out = torch.empty(need, dtype=torch.uint8, device=DEV), torch.empty_like(q)
    args = lambda p, n: (heads, tok, cache._cache(), 1.0, 0, out.data_ptr(), p, n, None)  # noqa: E731
    for p, n in ((ws.data_ptr(), need - 1), (None, need), (None, 0)):
        assert _abi.lib.ep_paged_attention(*args(p, n)) == -3 and _abi.last_error()
    assert _abi.lib.ep_paged_attention(*args(ws.data_ptr() + 8, need)) == 2


@pytest.mark.parametrize("dim", [64, 40])
def test_a_rotation_without_positions_has_no_tables(dim):
    """max_pos 0: the tables may be null, and every position lies past them."""
    g = gen(8)
    x, out = normal(g, 1, 3, 2, 64), torch.zeros(1, 3, 2, 64, dtype=BF16, device=DEV)
    pos = torch.tensor([[0, -1, 5]], device=DEV)
    heads = _abi.Heads(x.data_ptr(), _abi.BF16, 2, 384, 128, 64)
    tok = _abi.Tokens(1, 3, pos.data_ptr(), 3, 1, None, 0, 0)
    stream = _abi.stream_handle(DEV)
    assert _abi.lib.ep_rotate(heads, None, _abi.Rotation(None, None, 0, dim, 0), tok, 64, 0, out.data_ptr(), None,
                              stream) == 0
    assert out[0, [0, 2]].isnan().all() and (out[0, 1] == 0).all()


@pytest.mark.parametrize("length", [90, 3000])
@pytest.mark.parametrize("group", [2, 4])
@pytest.mark.parametrize("dim,dtype", [(64, F16), (96, BF16), (128, BF16), (192, F16), (256, BF16), (256, F16),
                                       (192, E4M3), (256, E4M3)])
def test_values_that_are_not_finite_reach_the_rows_and_columns_that_see_them(dim, dtype, group, length):
    """Eight tokens, 16 or 32 rows a key head; windows that begin and end
    around positions with an infinity or a NaN in a column of every four."""
    g = gen(9)
    qdt = dtype if dtype.itemsize == 2 else BF16
    pages = -(-length // 16)
    cache = epure.PagedKVCache(pages, 16, 2, dim, dtype, DEV)
    table = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)[None]
    pos = torch.arange(length, device=DEV)[None]
    k, v = normal(g, 1, length, 2, dim, dtype=F32), normal(g, 1, length, 2, dim, dtype=F32)
    v[0, length - 5, 0, 0::4] = float("inf")
    v[0, length - 3, 1, 3::4] = float("nan")
    v[0, length - 3, 0, dim - 1] = float("-inf")
    v[0, 22, :, 1::4] = float("nan")
    cache.append(k, v, pos, table)
    kc, vc = op.stands_for(k, dtype), op.stands_for(v, dtype)
    q = normal(g, 1, 8, 2 * group, dim, dtype=qdt)
    rows = torch.arange(length - 8, length, device=DEV)[None]
    window = length - 26                 # from 19 .. 26: the first four rows see 22
    out = cache.attend(q, rows, table, window=window).cpu()
    want, mag, big = op.attend(q, kc, vc, rows.cpu(), dim ** -0.5, window)
    clean = torch.isfinite(want)
    assert clean.any() and not clean.all()
    assert torch.equal(torch.isfinite(out), clean)
    tol = op.attend_tolerance(want, mag, big, qdt, dim)
    assert ((out.double() - want).abs() <= tol)[clean].all()


@pytest.mark.parametrize("dtype,qdt", [(BF16, BF16), (F16, F16), (I8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("S,group", [(1, 5), (2, 6), (3, 7)])
@pytest.mark.parametrize("D", [32, 112, 144, 160, 176, 208])
def test_head_sizes_between_powers_of_two(D, S, group, dtype, qdt):
    """What 16 lanes with 4, 8, 12 or 16 columns each cover, in part and whole."""
    g = gen(10)
    lengths = [1 + S, 200, 1700]
    cache, table, kc, vc = filled(g, lengths, 32, 2, D, dtype)
    pos = (torch.tensor(lengths, device=DEV)[:, None] - S + torch.arange(S, device=DEV))
    q = normal(g, 3, S, 2 * group, D, dtype=qdt)
    check(cache, table, q, pos, kc, vc)
    check(cache, table, q, pos, kc, vc, window=37)

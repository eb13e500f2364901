"""Rotary positions, the paged cache and attention over it on the GPU,
against the plain restatements of oracle/paged.py."""
import itertools

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


# ------------------------------------------------------------------ rotation
def rotate_tolerance(x, y, cos, m, dtype):
    """f32 tables, products and sum: each rounds once, half a step of at most
    m (|a| + |b|) together (3 * 2^-24); the output type's half step."""
    pair = x.detach().cpu().double().abs().amax(-1, keepdim=True) * 2 * m
    return op.half_step(y, dtype) + 3 * 2.0 ** -24 * pair


LAYOUTS = ["half", "interleaved"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("B,S,Hq,Hk,D,R", [(1, 1, 1, 1, 128, 128), (2, 7, 5, 1, 96, 64), (1, 33, 3, 2, 80, 40),
                                           (3, 2, 2, 2, 7, 2), (1, 5, 4, 4, 256, 256), (2, 3, 1, 1, 19, 18),
                                           (1, 2, 2, 1, 1040, 48)])
def test_rotation(B, S, Hq, Hk, D, R, dtype, layout):
    g = gen(B * S + D)
    q, k = normal(g, B, S, Hq, D, dtype=dtype), normal(g, B, S, Hk, D, dtype=dtype)
    scaling = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32}
    r = epure.Rotary(R, 50, theta=1e3, layout=layout, scaling=scaling, device=DEV)
    pos = torch.randint(-1, 52, (B, S), generator=g, device=DEV)
    got = r.rotate(q, k, pos)
    m = float(r.cos.abs().max())
    for x, y in zip((q, k), got):
        want = op.rotate(x, pos, r.cos, r.sin, layout == "interleaved")
        assert y.dtype == dtype and y.shape == x.shape
        bad = want.isnan()
        assert torch.equal(y.cpu().isnan(), bad)
        y, want = y.cpu().double()[~bad], want[~bad]
        tol = rotate_tolerance(x, op.rotate(x, pos, r.cos, r.sin, layout == "interleaved"), r.cos, m, dtype)[~bad]
        assert ((y - want).abs() <= tol).all()
    assert torch.equal(r(q, pos), got[0]) or got[0].isnan().any()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_rotation_of_strided_and_unaligned_inputs_is_the_same(layout):
    g = gen(4)
    r = epure.Rotary(64, 40, layout=layout, device=DEV)
    pos = torch.arange(9, device=DEV)
    q, k = normal(g, 2, 9, 4, 64), normal(g, 2, 9, 2, 64)
    want = r.rotate(q, k, pos)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)             # heads outside tokens
    pad = torch.empty(2, 9, 4, 67, dtype=BF16, device=DEV)         # odd strides, odd offset
    pad[..., 1:65] = q
    wide = torch.empty(2, 9, 2, 128, dtype=BF16, device=DEV)       # values two apart
    wide[..., ::2] = k
    for a, b in itertools.product((q, t, pad[..., 1:65]), (k, wide[..., ::2])):
        got = r.rotate(a, b, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = q[:, :, :1].expand(2, 9, 4, 64)                          # one head seen as four
    assert torch.equal(r(one, pos), r(q[:, :, :1], pos).expand(2, 9, 4, 64))
    for p in (pos.int(), pos.expand(2, 9), pos[None], torch.stack((pos, pos), 1).T):
        assert torch.equal(r.rotate(q, k, p)[0], want[0])


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("R", [64, 24])
def test_rotation_gradient(layout, R):
    """Against the formula (the turn the other way) and against differences
    of the forward pass: it is linear, so a difference of step 1 has no
    truncation error, only the rounding of the two sums (each value of y is
    off by 3 * 2^-24 of its pair, some 4 in magnitude)."""
    g = gen(6)
    r = epure.Rotary(R, 30, layout=layout, device=DEV)
    pos = torch.tensor([[3, 29, 0, -1]], device=DEV)
    q = normal(g, 1, 4, 3, 64, dtype=F32).requires_grad_()
    k = normal(g, 1, 4, 1, 64, dtype=F32).requires_grad_()
    gq, gk = normal(g, 1, 4, 3, 64, dtype=F32), normal(g, 1, 4, 1, 64, dtype=F32)
    y = r.rotate(q, k, pos)
    dq, dk = torch.autograd.grad(y, (q, k), (gq, gk))
    for d, up in ((dq, gq), (dk, gk)):
        want = op.rotate(up, pos, r.cos, r.sin, layout == "interleaved", inverse=True)
        assert ((d.cpu().double() - want).abs() <= rotate_tolerance(up, want, r.cos, 1.0, F32)).all()
    with torch.no_grad():
        for idx in [(0, 0, 0, 0), (0, 1, 2, R // 2), (0, 1, 1, R - 1), (0, 2, 0, 63), (0, 3, 1, 5)]:
            e = torch.zeros_like(q)
            e[idx] = 1.0
            diff = ((r(q + e, pos).double() - r(q, pos).double()) * gq.double()).sum().item()
            assert abs(diff - dq[idx].item()) <= 64 * 2.0 ** -24 * 16


def test_rotation_gradient_of_one_output_of_shared_heads_and_twice():
    g = gen(7)
    r = epure.Rotary(32, 30, device=DEV)
    pos = torch.arange(5, device=DEV)[None]
    q, k = normal(g, 1, 5, 2, 32, dtype=F32).requires_grad_(), normal(g, 1, 5, 1, 32, dtype=F32).requires_grad_()
    up = normal(g, 1, 5, 4, 32, dtype=F32)
    # keys shared by four heads; q's output unused
    _, y = r.rotate(q, k.expand(1, 5, 4, 32), pos)
    (y * up).sum().backward()
    assert q.grad is None
    want = op.rotate(up, pos, r.cos, r.sin, inverse=True).sum(2, keepdim=True)
    assert ((k.grad.cpu().double() - want).abs() <= 1e-5).all()    # 4 values of up to 5, 3 * 2^-24 each, and their sum
    k.grad = None
    y, _ = r.rotate(q, k.detach(), pos)
    (dq,) = torch.autograd.grad(y.sum(), q, retain_graph=True)     # an expanded upstream gradient
    want = op.rotate(torch.ones(1, 5, 2, 32), pos, r.cos, r.sin, inverse=True)
    assert (dq.cpu().double() - want).abs().max() <= 3 * 2.0 ** -23
    # the gradient is a turn of the upstream gradient w, and differentiable in it
    w, z = up[:, :, :2].clone().requires_grad_(), normal(g, 1, 5, 2, 32, dtype=F32)
    (dq,) = torch.autograd.grad((y * w).sum(), q, create_graph=True)
    (dw,) = torch.autograd.grad((dq * z).sum(), w)
    assert torch.equal(dw, r(z, pos))


def test_empty_rotations():
    r = epure.Rotary(32, 30, device=DEV)
    for shape in [(0, 3, 2, 32), (2, 0, 2, 32), (2, 3, 0, 32)]:
        x = torch.empty(shape, device=DEV)
        assert r(x, torch.zeros(shape[:2], dtype=torch.int64, device=DEV)).shape == shape


# ------------------------------------------------------------------ the cache
def table_of(g, need, page, n_pages):
    """A shuffled page table [B, W]; unused entries name no page."""
    rows = [(n + page - 1) // page for n in need]
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    t = torch.full((len(need), max(max(rows), 1)), -7, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(rows):
        t[b, :n] = order[at:at + n]
        at += n
    return t


def poison(cache):
    """NaN in every slot (and scale) that is not written."""
    for t in (cache.k, cache.v):
        if t.dtype.itemsize == 2:
            t.fill_(float("nan"))
        else:
            t.view(torch.uint8).fill_(0x7f)        # NaN in e4m3, 127 in int8
    for s in (cache.k_scale, cache.v_scale):
        if s is not None:
            s.fill_(float("nan"))


@pytest.mark.parametrize("dtype", [BF16, F16, E4M3, I8])
@pytest.mark.parametrize("xdt", [BF16, F32])
@pytest.mark.parametrize("page,H,D", [(16, 1, 64), (32, 3, 80), (64, 2, 128), (128, 1, 256), (16, 2, 16)])
def test_append_and_read(page, H, D, xdt, dtype):
    g = gen(page + D)
    need = [37, 1, 0, 20]
    cache = epure.PagedKVCache(9, page, H, D, dtype, DEV)
    poison(cache)
    before = cache.k.view(torch.uint8).clone()
    table = table_of(g, need, page, 9)
    pos = torch.arange(37, device=DEV).expand(4, 37).clone()
    for b, n in enumerate(need):
        pos[b, n:] = -1
    kv = normal(g, 4, 37, 2 * H, D, dtype=xdt, std=3.0)
    kv[0, 3], kv[0, 4, 0], kv[1, 0, :, 5] = 0.0, 2.0 ** -120, 1000.0
    k, v = kv[:, :, :H], kv[:, :, H:]
    assert cache.append(k, v, pos, table) is None
    out = cache.read(pos, table, F32)
    real = (pos >= 0).cpu()
    for x, y in zip((k, v), out):
        want = op.stands_for(x, dtype)
        assert torch.equal(y.cpu()[real], want[real]) and (y.cpu()[~real] == 0).all()
        for dt in (BF16, F16):
            assert torch.equal(cache.read(pos, table, dt)[0].cpu()[real], op.stands_for(k, dtype).to(dt)[real])
    used = torch.zeros(9, page, dtype=torch.bool)
    for b in range(4):
        for p in range(need[b]):
            used[int(table[b, p // page]), p % page] = True
    after = cache.k.view(torch.uint8).cpu().transpose(1, 2)
    assert torch.equal(after[~used], before.cpu().transpose(1, 2)[~used])      # nothing else was written


@pytest.mark.parametrize("dtype", [BF16, E4M3, I8])
def test_rows_with_infinities_or_nan(dtype):
    cache = epure.PagedKVCache(1, 16, 1, 64, dtype, DEV)
    x = normal(gen(1), 1, 4, 1, 64)
    x[0, 1, 0, 7], x[0, 2, 0, 63] = float("inf"), float("nan")
    pos, table = torch.arange(4, device=DEV)[None], torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    cache.append(x, x, pos, table)
    for y in cache.read(pos, table, F32):
        y = y.cpu()
        if dtype == BF16:
            assert torch.equal(y.nan_to_num(9.0), x.float().cpu().nan_to_num(9.0)) and y[0, 1, 0, 7] == float("inf")
        else:
            assert y[0, 1:3].isnan().all() and torch.isfinite(y[0, [0, 3]]).all()


@pytest.mark.parametrize("layout,R", [("half", 64), ("interleaved", 64), ("half", 40), ("interleaved", 26)])
@pytest.mark.parametrize("dtype", [F16, E4M3, I8])
def test_append_turns_q_and_k(dtype, layout, R):
    g = gen(R)
    cache = epure.PagedKVCache(4, 16, 2, 64, dtype, DEV)
    r = epure.Rotary(R, 30, layout=layout, device=DEV)
    q, k, v = (normal(g, 2, 13, h, 64, dtype=F16) for h in (6, 2, 2))
    pos, table = torch.arange(13, device=DEV).expand(2, 13) + 5, table_of(g, [18, 18], 16, 4)
    qo = cache.append(k, v, pos, table, q=q, rotary=r)
    assert torch.equal(qo, r(q, pos))
    ko, vo = cache.read(pos, table, F32)
    turned = op.rotate32(k, pos, r.cos, r.sin, layout == "interleaved")
    assert torch.equal(ko.cpu(), op.stands_for(turned, dtype)) and torch.equal(vo.cpu(), op.stands_for(v, dtype))
    # no rotation: q comes back as it went in; positions past the rotation's tables are not stored
    assert torch.equal(cache.append(k, v, pos, table, q=q), q)
    poison(cache)
    short = epure.Rotary(R, 10, layout=layout, device=DEV)
    qo = cache.append(k, v, pos, table, q=q, rotary=short)
    assert qo[:, 5:].isnan().all() and torch.isfinite(qo[:, :5]).all()
    ko, vo = cache.read(pos, table, F32)
    assert torch.isfinite(ko[:, :5]).all() and (dtype != I8 or ko[:, 5:].isnan().all())


def test_append_of_unaligned_rows_is_the_same():
    g = gen(12)
    table, pos = table_of(g, [9], 16, 2), torch.arange(9, device=DEV)[None]
    k = normal(g, 1, 9, 2, 80)
    pad = torch.empty(1, 9, 2, 83, dtype=BF16, device=DEV)
    pad[..., 1:81] = k
    r = epure.Rotary(80, 30, device=DEV)
    out = []
    for x in (k, pad[..., 1:81], torch.stack((k, k), -1)[..., 0]):
        cache = epure.PagedKVCache(2, 16, 2, 80, I8, DEV)
        out.append((cache.append(x, x, pos, table, q=x, rotary=r), cache.k, cache.v, cache.k_scale, cache.v_scale))
    for o in out[1:]:
        assert all(torch.equal(a, b) for a, b in zip(out[0], o))


def test_positions_and_pages_out_of_range_store_nothing_and_read_nan():
    cache = epure.PagedKVCache(3, 16, 1, 64, BF16, DEV)
    table = torch.tensor([[0, 3], [-1, 1], [2, 1 << 30]], dtype=torch.int32, device=DEV)
    pos = torch.tensor([[0, 16, 32, 1 << 40], [0, 16, -5, 31], [15, 16, 17, 31]], device=DEV)
    x = normal(gen(3), 3, 4, 1, 64)
    cache.append(x, x, pos, table)
    y = cache.read(pos, table)[0]
    ok = torch.tensor([[1, 0, 0, 0], [0, 1, 0, 1], [1, 0, 0, 0]], dtype=torch.bool, device=DEV)
    pad = pos < 0
    assert torch.equal(y[ok], x[ok]) and (y[pad] == 0).all() and y[~ok & ~pad].isnan().all()
    assert int((cache.k.view(torch.int16) != 0).any(-1).sum()) == 4
    out = cache.attend(x, pos, table)
    assert torch.equal(out.isnan().all(-1).squeeze(-1).cpu(),
                       torch.tensor([[0, 1, 1, 1], [1, 1, 0, 1], [0, 1, 1, 1]], dtype=torch.bool))


# ------------------------------------------------------------------ attention
def context(g, cache, table, lengths, xdt, std=1.0):
    """Random keys and values at positions 0 .. length - 1 of every sequence;
    returns what the cache holds of them, [B, L, heads, D] f32."""
    n = max(max(lengths), 1)
    pos = torch.arange(n, device=DEV).expand(len(lengths), n).clone()
    for b, m in enumerate(lengths):
        pos[b, m:] = -1
    k, v = (normal(g, len(lengths), n, cache.heads, cache.dim, dtype=xdt, std=std) for _ in range(2))
    cache.append(k, v, pos, table)
    return op.stands_for(k, cache.dtype), op.stands_for(v, cache.dtype)


def check_attend(cache, table, q, pos, kc, vc, **kw):
    out = cache.attend(q, pos, table, **kw)
    assert out.shape == q.shape and out.dtype == q.dtype
    want, mag, big = op.attend(q, kc, vc, pos.cpu(), kw.get("scale", cache.dim ** -0.5), kw.get("window"))
    tol = op.attend_tolerance(want, mag, big, q.dtype, cache.dim)
    err = (out.cpu().double() - want).abs()
    assert (err <= tol).all(), f"worst {(err / tol.clamp(min=1e-300)).max().item():.3g} of the tolerance"
    return out


TYPES = [(BF16, BF16), (F16, F16), (I8, BF16), (I8, F16), (E4M3, BF16), (E4M3, F16)]


@pytest.mark.parametrize("cdt,qdt", TYPES)
@pytest.mark.parametrize("D", [64, 80, 128, 192, 256, 16])
def test_attend_one_token_of_ragged_lengths(D, cdt, qdt):
    g = gen(D)
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300]
    cache = epure.PagedKVCache(64, 16, 2, D, cdt, DEV)
    poison(cache)
    table = table_of(g, lengths, 16, 64)
    kc, vc = context(g, cache, table, lengths, F32)
    q = normal(g, len(lengths), 1, 6, D, dtype=qdt, std=2.0)
    pos = torch.tensor(lengths, device=DEV)[:, None] - 1
    check_attend(cache, table, q, pos, kc, vc)


@pytest.mark.parametrize("cdt,qdt", [(BF16, BF16), (I8, F16), (E4M3, BF16)])
@pytest.mark.parametrize("G,S", [(1, 1), (4, 1), (16, 1), (17, 1), (5, 3), (8, 5), (1, 40), (3, 37)])
@pytest.mark.parametrize("window", [None, 1, 50])
def test_attend_several_tokens_groups_and_windows(G, S, window, cdt, qdt):
    g = gen(G * S)
    lengths = [200, S, max(S - 2, 0), 77]
    cache = epure.PagedKVCache(20, 32, 2, 64, cdt, DEV)
    poison(cache)
    table = table_of(g, lengths, 32, 20)
    kc, vc = context(g, cache, table, lengths, F32)
    q = normal(g, 4, S, 2 * G, 64, dtype=qdt, std=2.0)
    pos = torch.tensor(lengths, device=DEV)[:, None] - S + torch.arange(S, device=DEV)
    check_attend(cache, table, q, pos, kc, vc, window=window, scale=0.2)


@pytest.mark.parametrize("page", [16, 32, 64, 256, 1024])
@pytest.mark.parametrize("cdt,qdt", [(BF16, BF16), (I8, BF16)])
def test_attend_long_contexts_split_over_their_length(page, cdt, qdt):
    g = gen(page)
    lengths = [5000, 37, 2049]
    n = sum(-(-m // page) for m in lengths) + 1
    cache = epure.PagedKVCache(n, page, 1, 128, cdt, DEV)
    poison(cache)
    table = table_of(g, lengths, page, n)
    kc, vc = context(g, cache, table, lengths, F32)
    q = normal(g, 3, 1, 4, 128, dtype=qdt, std=3.0)
    pos = torch.tensor(lengths, device=DEV)[:, None] - 1
    check_attend(cache, table, q, pos, kc, vc)
    check_attend(cache, table, q, pos, kc, vc, window=1000)


def test_attend_in_any_order_of_positions_and_with_padding():
    """Rows need not be the newest tokens, nor in order."""
    g = gen(30)
    cache = epure.PagedKVCache(10, 16, 1, 64, BF16, DEV)
    table = table_of(g, [150], 16, 10)
    kc, vc = context(g, cache, table, [150], F32)
    pos = torch.tensor([[149, -1, 0, 100, 16, -1, 3]], device=DEV)
    q = normal(g, 1, 7, 2, 64, std=2.0)
    check_attend(cache, table, q, pos, kc, vc)
    check_attend(cache, table, q, pos, kc, vc, window=20)


@pytest.mark.parametrize("what", ["large scores", "equal scores", "negative scale", "large values"])
@pytest.mark.parametrize("qdt", [BF16, F16])
def test_attend_extreme_scores(what, qdt):
    g = gen(31)
    cache = epure.PagedKVCache(30, 16, 1, 64, qdt, DEV)
    table = table_of(g, [450], 16, 30)
    kc, vc = context(g, cache, table, [450], F32, std=100.0 if what == "large values" else 1.0)
    q = normal(g, 1, 1, 4, 64, dtype=qdt, std={"large scores": 50.0, "equal scores": 0.0}.get(what, 1.0))
    check_attend(cache, table, q, torch.tensor([[449]], device=DEV), kc, vc,
                 scale=-0.125 if what == "negative scale" else 0.125)


@pytest.mark.parametrize("cdt", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_masked_infinities_and_nan_do_not_reach_a_row(bad, cdt):
    """A row's later positions, and those before its window, may hold
    anything; a row that attends to them does get them."""
    g = gen(33)
    qdt = cdt if cdt.itemsize == 2 else BF16
    cache = epure.PagedKVCache(5, 16, 2, 64, cdt, DEV)
    table = table_of(g, [80], 16, 5)
    pos = torch.arange(80, device=DEV)[None]
    k, v = normal(g, 1, 80, 2, 64, dtype=F32), normal(g, 1, 80, 2, 64, dtype=F32)
    v[0, 70, :, 3], v[0, 40, :, 5] = bad, bad
    k[0, 71, :, 0] = bad
    cache.append(k, v, pos, table)
    kc, vc = op.stands_for(k, cdt), op.stands_for(v, cdt)
    q = normal(g, 1, 8, 4, 64, dtype=qdt)
    rows = torch.arange(66, 74, device=DEV)[None]
    out = cache.attend(q, rows, table, window=28).cpu()
    want, mag, big = op.attend(q, kc, vc, rows.cpu(), 0.125, 28)
    tol = op.attend_tolerance(want, mag, big, qdt, 64)
    clean = torch.isfinite(want)
    assert clean[0, 2:4].all() and not clean[0, :2, :, 5].any()          # 41 .. 69 only, and 40 among them
    assert ((out.double() - want).abs() <= tol)[clean].all()
    assert torch.equal(torch.isfinite(out), clean)
    early = cache.attend(q, rows - 30, table).cpu()          # positions 36 .. 43: 70 and 71 lie in later tiles
    want, mag, big = op.attend(q, kc, vc, (rows - 30).cpu(), 0.125)
    clean = torch.isfinite(want)
    assert clean[0, :4].all() and torch.equal(torch.isfinite(early), clean)
    assert ((early.double() - want).abs() <= op.attend_tolerance(want, mag, big, qdt, 64))[clean].all()


def test_attend_over_shared_pages_and_a_shared_table_row():
    """Two sequences with one prefix: their tables name the same pages."""
    g = gen(35)
    cache = epure.PagedKVCache(6, 32, 2, 64, BF16, DEV)
    one = table_of(g, [96], 32, 6)
    kc, vc = context(g, cache, one, [96], F32)
    q = normal(g, 3, 1, 4, 64)
    pos = torch.tensor([[95], [40], [64]], device=DEV)
    check_attend(cache, one.expand(3, -1), q, pos, kc.expand(3, -1, -1, -1), vc.expand(3, -1, -1, -1))


def test_attend_past_32_bit_offsets():
    """A pool of more than 2^32 bytes and 2^31 values a tensor."""
    page, heads, dim = 256, 8, 128
    n = (1 << 31) // (page * heads * dim) + 40
    g = gen(36)
    cache = epure.PagedKVCache(n, page, heads, dim, BF16, DEV)
    table = torch.arange(n - 1, n - 5, -1, dtype=torch.int32, device=DEV)[None]
    kc, vc = context(g, cache, table, [1000], F32)
    q = normal(g, 1, 1, 16, dim, std=2.0)
    check_attend(cache, table, q, torch.tensor([[999]], device=DEV), kc, vc)
    y = cache.read(torch.arange(1000, device=DEV)[None], table, F32)
    assert torch.equal(y[0].cpu(), kc) and torch.equal(y[1].cpu(), vc)
    del cache
    torch.cuda.empty_cache()


def test_attend_strided_queries_are_the_same():
    g = gen(37)
    cache = epure.PagedKVCache(8, 16, 2, 64, BF16, DEV)
    table = table_of(g, [60, 50], 16, 8)
    context(g, cache, table, [60, 50], F32)
    pos = torch.tensor([[57, 58, 59], [47, 48, 49]], device=DEV)
    q = normal(g, 2, 3, 4, 64)
    want = cache.attend(q, pos, table)
    qkv = torch.cat((q, normal(g, 2, 3, 4, 64)), 2)
    odd = torch.empty(2, 3, 4, 67, dtype=BF16, device=DEV)
    odd[..., 1:65] = q
    for x in (q.transpose(1, 2).contiguous().transpose(1, 2), qkv[:, :, :4], odd[..., 1:65],
              torch.stack((q, q), -1)[..., 1]):
        assert torch.equal(cache.attend(x, pos, table), want)
    assert torch.equal(cache.attend(q, pos.int(), table.repeat(1, 2)[:, ::1]), want)


def test_attend_twice_is_the_same():
    g = gen(38)
    cache = epure.PagedKVCache(300, 32, 2, 128, I8, DEV)
    lengths = [4000, 1, 1500, 900]
    table = table_of(g, lengths, 32, 300)
    context(g, cache, table, lengths, F32)
    q, pos = normal(g, 4, 1, 8, 128), torch.tensor(lengths, device=DEV)[:, None] - 1
    want = cache.attend(q, pos, table)
    for _ in range(5):
        assert torch.equal(cache.attend(q, pos, table), want)


def test_a_step_in_a_graph_and_on_another_stream():
    """Positions advance on the device; each replay equals the eager calls."""
    g = gen(39)
    B, H, D = 3, 2, 64
    r = epure.Rotary(D, 200, device=DEV)
    caches = [epure.PagedKVCache(24, 16, H, D, E4M3, DEV) for _ in range(2)]
    table = table_of(g, [100, 120, 90], 16, 24)
    start = torch.tensor([[60], [75], [0]], device=DEV)
    for c in caches:
        context(gen(40), c, table, [60, 75, 0], F32)
    q, k, v = (torch.zeros(B, 1, h, D, dtype=BF16, device=DEV) for h in (4, H, H))
    pos = start.clone()

    def step(c, p):
        return c.attend(c.append(k, v, p, table, q=q, rotary=r), p, table)

    steps = [[normal(g, *t.shape) for t in (q, k, v)] for _ in range(5)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0], pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(caches[0], pos)
        pos += 1
    pos.copy_(start)
    want_pos = start.clone()
    for vals in steps:
        for t, x in zip((q, k, v), vals):
            t.copy_(x)
        want = step(caches[1], want_pos)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        with torch.cuda.stream(side):
            again = caches[1].attend(r(q, want_pos), want_pos, table)
        torch.cuda.synchronize()
        assert torch.equal(again, want)
        want_pos += 1
    assert torch.equal(pos, want_pos)


def test_empty_calls():
    cache = epure.PagedKVCache(2, 16, 2, 64, BF16, DEV)
    for B, S in ((0, 1), (1, 0)):
        x = torch.empty(B, S, 2, 64, dtype=BF16, device=DEV)
        pos = torch.empty(B, S, dtype=torch.int64, device=DEV)
        table = torch.zeros(B, 1, dtype=torch.int32, device=DEV)
        assert cache.append(x, x, pos, table, q=x).shape == x.shape
        assert cache.attend(x, pos, table).shape == x.shape and cache.read(pos, table)[0].shape == x.shape
    x, pos = torch.ones(1, 1, 2, 64, dtype=BF16, device=DEV), torch.zeros(1, 1, dtype=torch.int64, device=DEV)
    none = torch.empty(1, 0, dtype=torch.int32, device=DEV)        # a table without pages
    cache.append(x, x, pos, none)
    assert cache.attend(x, pos, none).isnan().all() and (cache.attend(x, pos - 1, none) == 0).all()
    assert (cache.k == 0).all()


def test_refusals():
    cache = epure.PagedKVCache(2, 16, 2, 64, BF16, DEV)
    x, pos = torch.ones(2, 1, 2, 64, dtype=BF16, device=DEV), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    table = torch.zeros(2, 1, dtype=torch.int32, device=DEV)
    r = epure.Rotary(64, 4, device=DEV)
    value = [lambda: cache.append(x[:, :, :1], x, pos, table), lambda: cache.append(x, x, pos, table[:1]),
             lambda: cache.append(x, x, pos, table[0]), lambda: cache.append(x, x, pos, table, q=x[:1]),
             lambda: cache.append(x, x, torch.zeros(3, 1, dtype=torch.int64, device=DEV), table),
             lambda: cache.append(x.cpu(), x, pos, table), lambda: cache.append(x, x, pos.cpu(), table),
             lambda: cache.append(x, x, pos, table, rotary=epure.Rotary(128, 4, device=DEV)),
             lambda: cache.append(x, x, pos, table, rotary=epure.Rotary(64, 4, device="cpu")),
             lambda: cache.attend(x[..., :32], pos, table), lambda: cache.attend(x[:, :, :1], pos, table),
             lambda: cache.attend(x[0], pos, table), lambda: cache.attend(x, pos, table, window=0),
             lambda: cache.read(pos[0], table), lambda: r(x[..., :32], pos), lambda: r.rotate(x, x[:1], pos),
             lambda: r(x[0], pos)]
    types = [lambda: cache.append(x, x, pos.float(), table), lambda: cache.append(x, x, pos, table.long()),
             lambda: cache.append(x, x.float(), pos, table), lambda: cache.append(x.long(), x.long(), pos, table),
             lambda: cache.attend(x.float(), pos, table), lambda: cache.attend(x.half(), pos, table),
             lambda: cache.read(pos, table, torch.int8), lambda: r.rotate(x, x.float(), pos), lambda: r(x.int(), pos)]
    for call in value:
        with pytest.raises(ValueError):
            call()
    for call in types:
        with pytest.raises(TypeError):
            call()
    y = x.clone().requires_grad_()
    for call in (lambda: cache.attend(y, pos, table), lambda: cache.append(y, x, pos, table)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
        with torch.no_grad():
            call()

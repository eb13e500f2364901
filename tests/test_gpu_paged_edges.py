"""The paged operators where a call is out of the ordinary: tokens past the
rotation's tables, derivatives that only some tensors want, huge scores."""
import pytest
import torch
from torch.autograd import forward_ad

import epure
from epure.kernels import _abi, cuda
from oracle import paged as op

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    """Each call path of the operators."""
    assert _abi.call is not None, _abi.CALL_ERROR
    if request.param == "python":
        monkeypatch.setattr(_abi, "call", None)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def normal(g, *shape, dtype=BF16, std=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def raw(cache):
    """Everything that a cache holds, as bytes."""
    return [t.view(torch.uint8).clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]


# ------------------------------------------------------------------ past the rotation's tables
@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
@pytest.mark.parametrize("rot", [64, 40])
def test_a_token_past_the_rotations_tables_stores_neither_key_nor_value(dtype, rot, path):
    g = gen(1)
    r = epure.Rotary(rot, 10, device=DEV)
    q, k, v = (normal(g, 2, 13, h, 64) for h in (4, 2, 2))
    pos = torch.stack((torch.arange(13), 12 - torch.arange(13))).to(DEV)
    pos[0, 3] = -1
    table = torch.tensor([[2], [0]], dtype=torch.int32, device=DEV)
    caches = [epure.PagedKVCache(3, 16, 2, 64, dtype, DEV) for _ in range(3)]
    for c in caches:
        for t in (c.k, c.v):
            t.view(torch.uint8).fill_(0x5a)
    caches[0].append(k, v, torch.where(pos < 10, pos, -1), table, rotary=r)     # the rest as padding
    qo = caches[1].append(k, v, pos, table, q=q, rotary=r)
    assert caches[2].append(k, v, pos, table, rotary=r) is None
    past = pos >= 10
    assert qo[past].isnan().all() and not qo[~past].isnan().any()
    for c in caches[1:]:
        for a, b in zip(raw(caches[0]), raw(c)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------ windows
@pytest.mark.parametrize("window", [300, 2 ** 31, 2 ** 63 - 1, 2 ** 63, 2 ** 64 + 5, 2 ** 70])
def test_a_window_past_the_context_is_no_window(window, path):
    g = gen(2)
    cache = epure.PagedKVCache(20, 16, 1, 64, BF16, DEV)
    table = torch.randperm(20, generator=g, device=DEV).to(torch.int32)[None, :19]
    x, pos = normal(g, 1, 300, 1, 64), torch.arange(300, device=DEV)[None]
    cache.append(x, normal(g, 1, 300, 1, 64), pos, table)
    q = normal(g, 1, 2, 4, 64)
    assert torch.equal(cache.attend(q, pos[:, -2:], table, window=window), cache.attend(q, pos[:, -2:], table))


# ------------------------------------------------------------------ forward mode
def test_forward_mode_tangents_turn_with_the_values(path):
    """The turn is linear: its tangent is the tangent turned."""
    g = gen(3)
    r = epure.Rotary(48, 30, layout="interleaved", device=DEV)
    q, k, tq, tk = (normal(g, 2, 5, h, 64, dtype=F32) for h in (6, 2, 6, 2))
    pos = torch.tensor([[0, 5, 29, -1, 7]], device=DEV)
    want, turned = r.rotate(q, k, pos), r.rotate(tq, tk, pos)
    with forward_ad.dual_level():
        dq, dk = forward_ad.make_dual(q, tq), forward_ad.make_dual(k, tk)
        for a, b in ((dq, dk), (dq, k), (q, dk)):
            out = [forward_ad.unpack_dual(t) for t in r.rotate(a, b, pos)]
            for o, w, t, x, base in zip(out, want, turned, (a, b), (q, k)):
                assert torch.equal(o.primal, w)
                if x is base:
                    assert o.tangent is None or not o.tangent.any()
                else:
                    assert torch.equal(o.tangent, t)
        one = forward_ad.unpack_dual(r(dq, pos))
        assert torch.equal(one.primal, want[0]) and torch.equal(one.tangent, turned[0])
        with torch.no_grad():                       # which forward mode does not heed
            assert torch.equal(forward_ad.unpack_dual(r(dq, pos)).tangent, turned[0])
        # the tangent of a gradient: the upstream tangent turned back
        x = q.clone().requires_grad_()
        y = r(x, pos)
        (gt,) = torch.autograd.grad(r(x, pos), x, tq)
        try:
            (gx,) = torch.autograd.grad(y, x, forward_ad.make_dual(q, tq))
        except RuntimeError as e:                   # torch's C++ nodes have no forward mode, and say so
            assert "jvp" in str(e)
        else:
            assert torch.equal(forward_ad.unpack_dual(gx).tangent, gt)


def test_reverse_over_forward(path):
    g = gen(4)
    r = epure.Rotary(64, 30, device=DEV)
    q, tq, up = (normal(g, 1, 5, 2, 64, dtype=F32) for _ in range(3))
    pos = torch.arange(5, device=DEV)
    tq.requires_grad_()
    with forward_ad.dual_level():
        t = forward_ad.unpack_dual(r(forward_ad.make_dual(q, tq), pos)).tangent
        (got,) = torch.autograd.grad(t, tq, up)
    x = q.clone().requires_grad_()
    (want,) = torch.autograd.grad(r(x, pos), x, up)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ cache derivatives
def test_the_cache_refuses_what_it_has_no_derivative_for(path):
    g = gen(5)
    cache = epure.PagedKVCache(2, 16, 2, 64, BF16, DEV)
    x, pos = normal(g, 1, 3, 2, 64), torch.arange(3, device=DEV)[None]
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    leaf = normal(g, 2, 2, 16, 64).requires_grad_()
    held = epure.PagedKVCache.of(leaf, leaf.detach())
    before = raw(cache)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, x)
        dual = epure.PagedKVCache.of(leaf.detach(), forward_ad.make_dual(leaf.detach(), leaf.detach()))
        calls = [lambda: cache.append(d, x, pos, table), lambda: cache.append(x, d, pos, table),
                 lambda: cache.append(x, x, pos, table, q=d), lambda: cache.attend(d, pos, table),
                 lambda: dual.attend(x, pos, table), lambda: dual.read(pos, table),
                 lambda: held.attend(x, pos, table), lambda: held.read(pos, table)]
        for call in calls:
            with pytest.raises(RuntimeError, match="no backward|no derivative"):
                call()
    for a, b in zip(before, raw(cache)):
        assert torch.equal(a, b)
    with torch.no_grad():
        assert torch.equal(held.read(pos, table)[0].float(),
                           leaf.detach()[0, :, :3].transpose(0, 1)[None].float())


# ------------------------------------------------------------------ gradients of one of two
@pytest.mark.parametrize("which", [0, 1])
def test_only_what_wants_a_gradient_gets_one(which, path):
    """rotate(q, k) with one of them a leaf: the other's output is a constant,
    and the cache takes it."""
    g = gen(6)
    r = epure.Rotary(64, 30, device=DEV)
    xs = [normal(g, 1, 5, h, 64) for h in (4, 2)]
    ups = [normal(g, 1, 5, h, 64) for h in (4, 2)]
    xs[which].requires_grad_()
    pos = torch.arange(5, device=DEV)[None]
    y = r.rotate(*xs, pos)
    assert y[which].requires_grad and not y[1 - which].requires_grad
    (got,) = torch.autograd.grad(y[which], xs[which], ups[which])
    both = [x.detach().requires_grad_() for x in xs]
    want = torch.autograd.grad(r.rotate(*both, pos), both, ups)[which]
    assert torch.equal(got, want)
    for a, b in zip(y, r.rotate(*(x.detach() for x in xs), pos)):
        assert torch.equal(a, b)
    if which == 0:
        cache = epure.PagedKVCache(1, 16, 2, 64, BF16, DEV)
        cache.append(y[1], ups[1], pos, torch.zeros(1, 1, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------ two tensors
def test_rotate_wants_two_tensors(path):
    r = epure.Rotary(64, 30, device=DEV)
    x, pos = normal(gen(7), 1, 5, 2, 64), torch.arange(5, device=DEV)
    for q in (x, x.clone().requires_grad_()):
        for a, b in ((q, None), (None, q)):
            with pytest.raises(TypeError):
                r.rotate(a, b, pos)


# ------------------------------------------------------------------ no heads
@pytest.mark.parametrize("heads", [(0, 2), (2, 0), (0, 0)])
@pytest.mark.parametrize("grad", [False, True])
def test_one_of_two_tensors_without_heads(heads, grad, path):
    r = epure.Rotary(64, 30, device=DEV)
    g = gen(8)
    x = [normal(g, 1, 5, h, 64).requires_grad_(grad) for h in heads]
    pos = torch.arange(5, device=DEV)
    y = r.rotate(*x, pos)
    for a, b in zip(x, y):
        assert b.shape == a.shape and (a.shape[2] == 0 or torch.equal(b, r(a, pos)))
    if grad:
        for a, d in zip(x, torch.autograd.grad(y, x, [torch.ones_like(t) for t in y])):
            assert d.shape == a.shape


# ------------------------------------------------------------------ a call of one and of two
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("rot", [64, 40])
def test_one_tensor_turns_as_two_do_past_the_tables_too(layout, rot, path):
    g = gen(9)
    r = epure.Rotary(rot, 20, layout=layout, device=DEV)
    q, k = normal(g, 2, 6, 3, 64), normal(g, 2, 6, 1, 64)
    pos = torch.tensor([[0, 19, 20, -1, 5, 1 << 40]], device=DEV).expand(2, 6)
    for x, y in zip((q, k), r.rotate(q, k, pos)):
        one = r(x, pos)
        assert torch.equal(one.view(torch.int16), y.view(torch.int16))
        assert torch.equal(one.isnan().all(-1).all(-1), pos >= 20) and torch.equal(one.isnan().any(-1).any(-1), pos >= 20)


# ------------------------------------------------------------------ huge scores
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("length", [1, 33, 2000])
def test_huge_f16_scores_keep_their_weights(length, sign):
    """Equal scores of up to 2^28 either way: each position weighs 1 /
    length, whatever the score's last bits are.  Keys of one sequence are
    equal, so its scores are, bit for bit."""
    g = gen(10)
    B, D = 3, 64
    pages = -(-length // 16)
    cache = epure.PagedKVCache(B * pages, 16, 1, D, F16, DEV)
    table = torch.randperm(B * pages, generator=g, device=DEV).to(torch.int32).view(B, pages)
    pos = torch.arange(length, device=DEV).expand(B, -1)
    k = torch.randint(1000, 3000, (B, 1, 1, D), generator=g, device=DEV).to(F16).expand(B, length, 1, D)
    v = normal(g, B, length, 1, D, dtype=F16)
    cache.append(k, v, pos, table)
    q = torch.randint(20, 8000, (B, 1, 16, 1), generator=g, device=DEV).to(F16).expand(B, 1, 16, D).contiguous()
    out = cache.attend(q, pos[:, -1:], table, scale=sign * 0.125).cpu().double()
    want = v.cpu().double().mean(1, keepdim=True).expand(B, 1, 16, D)
    mag = v.cpu().double().abs().mean(1, keepdim=True).expand(B, 1, 16, D)
    assert ((out - want).abs() <= op.attend_tolerance(want, mag, 0.0, F16, D)).all()

"""Paged operators without a GPU: the oracle against brute force, the
frequencies of the scalings, the host-side checks of the classes and of the
C ABI (no launch is reached, so dummy pointers are never read)."""
import ctypes
import math

import pytest
import torch

import epure
from epure.kernels import _abi
from oracle import paged as op

E4M3 = torch.float8_e4m3fn


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("interleaved", [False, True])
def test_oracle_rotation_is_a_complex_product(interleaved):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2, 5, 3, 12, generator=g, dtype=torch.float64)
    t = torch.arange(9, dtype=torch.float64)[:, None] * torch.tensor([1.0, 0.3, 0.01, 1e-3])
    pos = torch.tensor([[0, 8, 3, -1, 9], [1, 2, 3, 4, 5]])
    y = op.rotate(x, pos, t.cos(), t.sin(), interleaved)
    r = x[..., :8]
    z = torch.complex(r[..., 0::2], r[..., 1::2]) if interleaved else torch.complex(r[..., :4], r[..., 4:])
    w = z * torch.polar(torch.ones(()).double(), t[pos.clamp(0, 8)])[:, :, None, :]
    want = torch.stack((w.real, w.imag), -1).flatten(-2) if interleaved else torch.cat((w.real, w.imag), -1)
    ok = (pos >= 0) & (pos < 9)
    assert torch.allclose(y[ok][..., :8], want[ok], atol=1e-14) and torch.equal(y[ok][..., 8:], x[ok][..., 8:])
    assert (y[0, 3] == 0).all() and y[0, 4].isnan().all()
    back = op.rotate(y, pos, t.cos(), t.sin(), interleaved, inverse=True)
    assert torch.allclose(back[ok], x[ok], atol=1e-14)


def test_oracle_codes_are_the_nearest_representable_values():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(40, 16, generator=g) * torch.exp2(torch.randint(-30, 30, (40, 1), generator=g).float())
    x[0] = 0.0
    x[1, :] = 0.0
    x[1, 3] = 448.0
    codes, scale = op.held(x, E4M3)
    values = torch.arange(256, dtype=torch.uint8).view(E4M3).float()
    values = values[torch.isfinite(values)]
    near = (x[..., None] / scale[..., None] - values).abs().amin(-1)
    assert torch.equal((x / scale - codes).abs(), near) and codes.abs().max() <= 448
    assert (codes[2:].abs().amax(-1) > 224 * (1 - 2.0 ** -5)).all()     # the least exponent that fits
    codes, scale = op.held(x, torch.int8)
    assert torch.equal(codes, codes.round()) and codes.abs().max() == 127
    assert ((codes * scale - x).abs() <= scale * (0.5 + 2.0 ** -15)).all()
    x[2, 5], x[3, 0] = math.inf, math.nan
    for dt in (E4M3, torch.int8):
        y = op.stands_for(x, dt)
        assert y[2:4].isnan().all() and torch.isfinite(y[4:]).all() and (y[0] == 0).all()


def test_oracle_attention_is_a_softmax_over_the_listed_positions():
    g = torch.Generator().manual_seed(3)
    q = torch.randn(1, 2, 4, 8, generator=g)
    k, v = torch.randn(1, 9, 2, 8, generator=g), torch.randn(1, 9, 2, 8, generator=g)
    k[0, 8], v[0, 8] = math.nan, math.nan          # after every row: not touched
    pos = torch.tensor([[6, -1]])
    o, mag, _ = op.attend(q, k, v, pos, 0.5, window=3)
    js = [4, 5, 6]
    for h in range(4):
        s = torch.stack([(q[0, 0, h] * k[0, j, h // 2]).sum() * 0.5 for j in js]).double()
        w = s.exp() / s.exp().sum()
        want = sum(w[i] * v[0, j, h // 2].double() for i, j in enumerate(js))
        assert torch.allclose(o[0, 0, h], want, atol=1e-6)
    assert (o[0, 1] == 0).all() and (mag >= o.abs() - 1e-12).all()


# ------------------------------------------------------------------ frequencies
def test_default_and_linear_frequencies():
    f, m = epure.rope_frequencies(8, 1e4)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    f2, _ = epure.rope_frequencies(8, 1e4, {"rope_type": "linear", "factor": 4.0})
    assert torch.equal(f2, f / 4)


def test_llama3_frequencies_keep_fast_pairs_and_divide_slow_ones():
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    f, _ = epure.rope_frequencies(128, 5e5)
    s, m = epure.rope_frequencies(128, 5e5, sc)
    turns = 8192 * f / (2 * math.pi)
    assert m == 1.0
    assert torch.equal(s[turns > 4], f[turns > 4]) and torch.allclose(s[turns < 1], f[turns < 1] / 8, rtol=1e-15)
    for i in ((turns >= 1) & (turns <= 4)).nonzero().flatten().tolist():
        a = (turns[i].item() - 1.0) / 3.0
        assert math.isclose(s[i].item(), (1 - a) * f[i].item() / 8 + a * f[i].item(), rel_tol=1e-12)
    assert (s[1:] < s[:-1]).all()


def test_yarn_frequencies_blend_between_two_pairs():
    sc = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    f, _ = epure.rope_frequencies(128, 1e4)
    s, m = epure.rope_frequencies(128, 1e4, sc)
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    assert torch.equal(s[:20], f[:20]) and torch.allclose(s[-10:], f[-10:] / 4, rtol=1e-15)
    ratio = s / f
    assert (ratio[1:] <= ratio[:-1] + 1e-15).all() and ratio.min() >= 0.25
    assert epure.rope_frequencies(128, 1e4, {**sc, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("scaling", [{"rope_type": "dynamic", "factor": 2.0}, {"rope_type": "linear", "factor": 0.0},
                                     {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 4.0,
                                      "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}])
def test_unserved_scalings_raise(scaling):
    with pytest.raises(ValueError):
        epure.rope_frequencies(64, 1e4, scaling)


def test_tables_hold_the_cosines_of_far_positions():
    r = epure.Rotary(64, 131072, theta=5e5, device="cpu")
    f, _ = epure.rope_frequencies(64, 5e5)
    for p in (0, 1, 65535, 65536, 131071):
        for i in (0, 5, 31):
            t = p * f[i].item()
            assert abs(r.cos[p, i].item() - math.cos(t)) <= 2.0 ** -24
            assert abs(r.sin[p, i].item() - math.sin(t)) <= 2.0 ** -24


# ------------------------------------------------------------------ refusals of the classes
@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(max_pos=0), dict(layout="quarter")])
def test_rotary_refuses(kw):
    with pytest.raises(ValueError):
        epure.Rotary(**{**dict(dim=8, max_pos=4, device="cpu"), **kw})


@pytest.mark.parametrize("page", [0, 8, 24, 2048])
def test_cache_refuses_page_sizes(page):
    with pytest.raises(ValueError):
        epure.PagedKVCache(2, page, 1, 64, device="cpu")


@pytest.mark.parametrize("dim", [8, 72, 272])
def test_cache_refuses_head_sizes(dim):
    with pytest.raises(ValueError):
        epure.PagedKVCache(2, 16, 1, dim, device="cpu")


def test_cache_refuses_types_and_mismatched_tensors():
    with pytest.raises(TypeError):
        epure.PagedKVCache(2, 16, 1, 64, dtype=torch.float32, device="cpu")
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(k, k[:1])
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(k, k, torch.ones(2, 1, 16), torch.ones(2, 1, 16))
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(k.to(torch.int8), k.to(torch.int8))
    with pytest.raises(ValueError):
        epure.PagedKVCache.of(k.view(2, 1, 64, 16).transpose(2, 3), k.view(2, 1, 64, 16).transpose(2, 3))
    c = epure.PagedKVCache.of(k, k.clone())
    assert (c.n_pages, c.heads, c.page, c.dim) == (2, 1, 16, 64)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the GPU tests cover the calls")
def test_calls_without_a_gpu_raise():
    r, c = epure.Rotary(8, 4, device="cpu"), epure.PagedKVCache(2, 16, 1, 64, device="cpu")
    x, pos = torch.zeros(1, 1, 1, 64), torch.zeros(1, 1, dtype=torch.int64)
    table = torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: r(x, pos), lambda: c.append(x, x, pos, table), lambda: c.read(pos, table),
                 lambda: c.attend(x.bfloat16(), pos, table)):
        with pytest.raises(RuntimeError, match="not available"):
            call()


# ------------------------------------------------------------------ refusals of the C ABI
P = 64      # a non-null, aligned address that no host check dereferences


def heads(n=4, dtype=_abi.BF16, ptr=P, d=64):
    return _abi.Heads(ptr, dtype, n, n * d, n * d, d)


def tokens(B=2, S=1, table=P, positions=P):
    return _abi.Tokens(B, S, positions, S, 1, table, 4, 4)


def cache(dtype=_abi.BF16, heads=2, page=16, D=64, n_pages=4, scales=None):
    s = scales if scales is not None else (P if dtype in (_abi.E4M3, _abi.I8) else None)
    return _abi.KVCache(P, P, s or None, s or None, dtype, heads, page, D, n_pages)


def rotation(dim=64):
    return _abi.Rotation(P, P, 16, dim, 0)


@pytest.fixture(scope="module")
def lib():
    assert _abi._load() is not None, _abi.LOAD_ERROR
    return _abi.lib


DTYPE, SHAPE, ARG = 1, 2, -1


@pytest.mark.parametrize("want,kw", [
    (ARG, dict(q=heads(0))), (DTYPE, dict(q=heads(dtype=_abi.E4M3))), (ARG, dict(q=heads(ptr=None))),
    (ARG, dict(k=heads(dtype=_abi.F16))), (ARG, dict(rot=rotation(63))), (ARG, dict(rot=rotation(0))),
    (ARG, dict(rot=rotation(128))), (ARG, dict(tok=tokens(positions=None))), (ARG, dict(tok=tokens(B=-1))),
    (SHAPE, dict(tok=tokens(B=1 << 20, S=1 << 20))), (SHAPE, dict(D=8192)), (ARG, dict(out=None))])
def test_rotate_rejects(lib, want, kw):
    a = dict(q=heads(), k=heads(2), rot=rotation(), tok=tokens(), D=64, out=P)
    a.update(kw)
    rc = lib.ep_rotate(a["q"], a["k"], a["rot"], a["tok"], a["D"], 0, a["out"], a["out"], None)
    assert rc == want and _abi.last_error()


CACHES = [(ARG, cache(heads=0)), (ARG, cache(n_pages=0)), (DTYPE, cache(dtype=_abi.F32)), (SHAPE, cache(page=8)),
          (SHAPE, cache(page=48)), (SHAPE, cache(page=2048)), (SHAPE, cache(D=72)), (SHAPE, cache(D=272)),
          (ARG, cache(dtype=_abi.I8, scales=0)), (ARG, cache(dtype=_abi.E4M3, scales=8))]


@pytest.mark.parametrize("want,c", CACHES)
def test_cache_calls_reject_the_cache(lib, want, c):
    assert lib.ep_kv_append(None, heads(2), heads(2), None, tokens(), c, None, None) == want
    assert lib.ep_kv_read(tokens(), c, P, P, _abi.BF16, None) == want
    assert lib.ep_paged_attention(heads(), tokens(), c, 1.0, 0, P, None, 0, None) == want
    assert lib.ep_paged_attention_workspace(heads(), tokens(), c) == 0


@pytest.mark.parametrize("want,kw", [
    (ARG, dict(k=heads(3))), (ARG, dict(v=heads(3))), (ARG, dict(v=heads(2, _abi.F16))),
    (ARG, dict(q=heads(4, _abi.F16))), (ARG, dict(q=heads(4))), (ARG, dict(rot=rotation(80))),
    (ARG, dict(tok=tokens(table=None))), (DTYPE, dict(k=heads(2, _abi.I8)))])
def test_append_rejects(lib, want, kw):
    a = dict(q=None, k=heads(2), v=heads(2), rot=None, tok=tokens())
    a.update(kw)
    assert lib.ep_kv_append(a["q"], a["k"], a["v"], a["rot"], a["tok"], cache(), None, None) == want


@pytest.mark.parametrize("want,kw", [
    (DTYPE, dict(q=heads(dtype=_abi.F32))), (DTYPE, dict(q=heads(dtype=_abi.F16))), (ARG, dict(q=heads(3))),
    (SHAPE, dict(q=heads(ptr=P + 8))), (SHAPE, dict(q=heads(d=60))), (ARG, dict(out=None)),
    (ARG, dict(tok=tokens(table=None)))])
def test_attention_rejects(lib, want, kw):
    a = dict(q=heads(), tok=tokens(), out=P)
    a.update(kw)
    assert lib.ep_paged_attention(a["q"], a["tok"], cache(), 1.0, 0, a["out"], None, 0, None) == want


def test_read_rejects(lib):
    assert lib.ep_kv_read(tokens(), cache(), P, P, _abi.I8, None) == DTYPE
    assert lib.ep_kv_read(tokens(), cache(), None, P, _abi.F32, None) == ARG


def test_descriptors_have_the_headers_sizes():
    assert ctypes.sizeof(_abi.Heads) == 40 and ctypes.sizeof(_abi.Tokens) == 64
    assert ctypes.sizeof(_abi.KVCache) == 56 and ctypes.sizeof(_abi.Rotation) == 32

"""The native call path of the paged operators (csrc/torch_paged.cpp): the
same results as the path through Python, and NotImplemented for what that
path has to check or refuse."""
import os
import subprocess

import pytest
import torch

import epure
from epure.kernels import _abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F16, F32, I8, E4M3 = torch.bfloat16, torch.float16, torch.float32, torch.int8, torch.float8_e4m3fn
DEV = torch.device("cuda:0")


def test_extension_is_rebuilt_with_the_paged_header():
    csrc = os.path.join(ROOT, "epure-runtime_amd", "csrc")
    out = os.path.abspath(_abi.TORCH_PATH)
    r = subprocess.run(["make", "-n", "-C", csrc, "-o", "torch_call.cpp", "-o", "torch_paged.cpp", "-o",
                        os.path.join(ROOT, "epure-runtime_amd", "_build", "torch_id"),
                        "-W", os.path.join(ROOT, "include", "epure_paged.h"), out],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "torch_paged.cpp" in r.stdout, r.stdout + r.stderr


def test_host_tensors_are_left_to_the_python_path():
    assert _abi._load() is not None and _abi.call is not None, (_abi.LOAD_ERROR, _abi.CALL_ERROR)
    x, pos = torch.zeros(1, 1, 1, 64, dtype=BF16), torch.zeros(1, 1, dtype=torch.int64)
    table, c, t = torch.zeros(1, 1, dtype=torch.int32), torch.zeros(2, 1, 16, 64, dtype=BF16), torch.zeros(4, 32)
    calls = [lambda: _abi.call.rotate(x, x, pos, t, t, False), lambda: _abi.call.rotate(x, None, pos, t, t, True),
             lambda: _abi.call.append(x, x, pos, table, None, None, None, False, c, c, None, None),
             lambda: _abi.call.read(pos, table, BF16, c, c, None, None),
             lambda: _abi.call.attend(x, pos, table, None, None, c, c, None, None)]
    for call in calls:
        assert call() is NotImplemented
    for call in (_abi.call.rotate, _abi.call.append, _abi.call.read, _abi.call.attend):
        with pytest.raises(TypeError):
            call(x)


# ------------------------------------------------------------------ on the GPU
gpu = pytest.mark.gpu


def normal(g, *shape, dtype=BF16):
    return torch.randn(*shape, generator=g, device=DEV).to(dtype)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture
def both(monkeypatch):
    """Runs f with the native path and without it."""
    def run(f):
        assert _abi.call is not None, _abi.CALL_ERROR
        native = f()
        with monkeypatch.context() as m:
            m.setattr(_abi, "call", None)
            plain = f()
        return native, plain
    return run


def same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert (x is None) == (y is None)
        if x is not None:
            assert x.dtype == y.dtype and x.shape == y.shape
            assert torch.equal(x.nan_to_num(7.0).float(), y.nan_to_num(7.0).float())


@gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_rotations_and_their_gradients_are_the_same(both, layout, dtype):
    g = gen(1)
    r = epure.Rotary(48, 30, layout=layout, device=DEV)
    q, k = normal(g, 2, 5, 6, 64, dtype=dtype), normal(g, 2, 5, 2, 64, dtype=dtype)
    up = normal(g, 2, 5, 6, 64, dtype=dtype), normal(g, 2, 5, 2, 64, dtype=dtype)
    wide = torch.cat((q, k), 2)
    poss = [torch.arange(5, device=DEV), torch.arange(5, device=DEV)[None],
            torch.tensor([[3], [-1]], device=DEV), torch.tensor(4, device=DEV),
            torch.tensor([[0, 1, 29, 30, -1], [7, 7, 7, 2, 1]], device=DEV)]

    def grads(a, b, pos):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = r.rotate(a, b, pos)
        ga, gb = torch.autograd.grad(y, (a, b), up, retain_graph=True)
        (only,) = torch.autograd.grad(y[1], b, up[1], retain_graph=True)
        (one,) = torch.autograd.grad(r(a, pos), a, up[0].transpose(0, 1).contiguous().transpose(0, 1))
        w = up[0].detach().requires_grad_()
        (ga2,) = torch.autograd.grad(y[0], a, w, create_graph=True)
        (dw,) = torch.autograd.grad(ga2, w, torch.ones_like(ga2))
        return [t.detach() for t in (*y, ga, gb, only, one, dw)]

    for pos in poss:
        for a, b in ((q, k), (wide[:, :, :6], wide[:, :, 6:])):
            same(*both(lambda: [*r.rotate(a, b, pos), r(a, pos)]))
            same(*both(lambda: grads(a, b, pos)))
    mixed = both(lambda: [t.detach() for t in r.rotate(q, k.detach().requires_grad_(), poss[0])])
    same(*mixed)


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16, I8, E4M3])
def test_cache_calls_are_the_same(both, dtype):
    g = gen(2)
    xdt = dtype if dtype.itemsize == 2 else BF16
    r = epure.Rotary(64, 60, device=DEV)
    q, k, v = (normal(g, 3, 4, h, 64, dtype=xdt) for h in (6, 2, 2))
    table = torch.randperm(12, generator=g, device=DEV).to(torch.int32).view(3, 4)
    pos = torch.tensor([[0, 1, 2, 3], [17, 18, 19, -1], [40, 63, 64, 5]], device=DEV)

    def calls():
        c = epure.PagedKVCache(12, 16, 2, 64, dtype, DEV)
        out = [c.append(k, v, pos, table), c.append(k, v, pos, table, q=q), c.append(k, v, pos, table, q=q, rotary=r),
               c.append(k, v, pos[:1], table[:, :2], rotary=r)]
        for dt in (F32, F16, BF16):
            out += c.read(pos, table, dt)
        out += [c.attend(q, pos, table), c.attend(q, pos, table, scale=0.3, window=3), c.attend(q, pos, table[:, ::2])]
        return out + [t.float() for t in (c.k, c.v)] + [c.k_scale, c.v_scale]

    same(*both(calls))


@gpu
def test_calls_under_a_torch_mode_or_of_subclasses_are_the_same():
    g = gen(3)
    r = epure.Rotary(64, 60, device=DEV)
    x, pos = normal(g, 1, 3, 2, 64), torch.arange(3, device=DEV)
    want = r(x, pos)
    p = torch.nn.Parameter(x)
    with torch.no_grad():
        assert torch.equal(r(p, pos), want)
    assert r(p, pos).requires_grad

    class Sub(torch.Tensor):
        pass
    got = r(x.as_subclass(Sub), pos)
    assert torch.equal(got.as_subclass(torch.Tensor), want)


@gpu
def test_a_gradient_captured_into_a_graph_replays():
    """The backward pass under capture, on the capture's stream."""
    g = gen(4)
    r = epure.Rotary(64, 60, device=DEV)
    q, k = (normal(g, 1, 8, h, 64, dtype=F32).requires_grad_() for h in (4, 2))
    up = [torch.zeros_like(q), torch.zeros_like(k)]
    pos = torch.arange(8, device=DEV)

    def grads():
        return torch.autograd.grad(r.rotate(q, k, pos), (q, k), up)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = grads()
    for _ in range(3):
        for t in up:
            t.copy_(normal(g, *t.shape, dtype=F32))
        want = [r(t, pos) for t in up]      # eager work between the replays
        graph.replay()
        torch.cuda.synchronize()
        same(out, grads())
        assert len(want) == 2

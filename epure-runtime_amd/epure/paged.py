"""Batches of sequences between the packed linears: rotary positions, a paged
key-value cache that is quantised as it is written, and attention of new
tokens over it, on the gfx950 kernels (include/epure_paged.h).

The reference leaves these to transformers (epure/runtime.py:373-415);
``epure.decode`` fuses them into one sequence's step.  Here every call takes
tokens as ``[B, S]`` (B sequences, S new tokens each): ``positions`` is an
integer tensor of their positions, ``table`` an int32 tensor ``[B, W]`` of the
pages that hold each sequence, ``table[b, i]`` the page of positions
``i * page .. (i + 1) * page - 1``.

Positions and pages are read on the device, so no call synchronizes and every
call can be captured in a HIP graph.  A negative position marks a padded
token: nothing is stored for it and its output row is zeros.  A position past
the rotation's or the table's range, or on a page that the pool lacks, stores
nothing and gives NaN rows.  GPU tensors only; what a kernel does not serve
raises.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad

from .kernels import _abi
from .kernels import cuda as cuda_kernel


def _require(*tensors):
    if not cuda_kernel.available():
        raise RuntimeError("the gfx950 HIP backend is not available")
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda or t.device != dev:
            raise ValueError(f"expected tensors on one GPU, got {[str(t.device) for t in tensors]}")
    return dev


def _no_grad(*tensors):
    for t in tensors:
        gradient, tangent = (False, False) if t is None else _wants(t)
        if gradient:
            raise RuntimeError("the paged cache has no backward: call under torch.no_grad()")
        if tangent:
            raise RuntimeError("the paged cache has no derivative: call it on tensors without tangents")


def _wants(t):
    """(a gradient, a forward-mode tangent): what is to be derived through t."""
    return torch.is_grad_enabled() and t.requires_grad, forward_ad.unpack_dual(t).tangent is not None


def _native():
    """The native call path, or None.  Its calls return NotImplemented for all
    that is not an ordinary call on plain GPU tensors: those go on below, where
    arguments are checked and refused."""
    return _abi.call if cuda_kernel.available() else None


def _run(what, rc):
    if not _abi.check(rc, what):
        raise ValueError(f"{what} declined: {_abi.last_error()}")


def _heads4(name, t):
    if t.dim() != 4:
        raise ValueError(f"{name} must be [B, S, heads, D], got {tuple(t.shape)}")
    if _abi.dtype_code(t.dtype) is None:
        raise TypeError(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _heads(t):
    return _abi.Heads(t.data_ptr(), _abi.dtype_code(t.dtype), t.shape[2], t.stride(0), t.stride(1), t.stride(2))


def _tokens(x, positions, table=None):
    """The tokens' descriptor for x's [B, S] and the tensors that it points at."""
    B, S = x
    if positions.dtype != torch.int64:
        if positions.dtype.is_floating_point or positions.dtype == torch.bool:
            raise TypeError(f"positions must be integers, got {positions.dtype}")
        positions = positions.to(torch.int64)
    if tuple(positions.shape) != (B, S):
        try:
            positions = positions.expand(B, S)
        except RuntimeError:
            raise ValueError(f"positions {tuple(positions.shape)} do not broadcast to [{B}, {S}]") from None
    t = _abi.Tokens(B, S, positions.data_ptr(), positions.stride(0), positions.stride(1), None, 0, 0)
    if table is not None:
        if table.dtype != torch.int32:
            raise TypeError(f"the page table must be int32, got {table.dtype}")
        if table.dim() != 2 or table.shape[0] != B:
            raise ValueError(f"the page table must be [{B}, pages], got {tuple(table.shape)}")
        if table.stride(1) != 1 and table.shape[1] > 1:
            table = table.contiguous()
        t.table, t.table_stride, t.width = table.data_ptr(), table.stride(0), table.shape[1]
    return t, (positions, table)


# Keys of a scaling that some kind reads, or that say nothing about the
# frequencies of ``dim`` rotated values (dim is the rotated part already).
_SCALING_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "factor",
                 "original_max_position_embeddings", "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow",
                 "attention_factor", "mscale", "mscale_all_dim", "truncate"}


def rope_frequencies(dim, theta=None, scaling=None):
    """Angle per position of the dim / 2 pairs (float64) and the attention factor.

    ``theta`` defaults to the scaling's ``rope_theta``, or 10000; both given
    have to agree.  ``scaling`` follows the models' configuration: a dict whose ``rope_type``
    is "default", "linear" (``factor``), "llama3" (``factor``,
    ``low_freq_factor``, ``high_freq_factor``,
    ``original_max_position_embeddings``: frequencies of fewer turns within
    the original context than ``low`` are divided by the factor, those of
    more than ``high`` kept, those between blended) or "yarn" (``factor``,
    ``original_max_position_embeddings``, ``beta_fast`` 32, ``beta_slow`` 1:
    the blend is linear in the pair's index between the pairs that make
    ``beta_fast`` and ``beta_slow`` turns, widened to whole indices unless
    ``truncate`` is false; the attention factor is ``attention_factor``, or
    M(mscale) / M(mscale_all_dim) with both given, or M(1), where M(s) = 0.1 s
    ln(factor) + 1, and 1 for factors up to 1).  A key that none of them knows
    raises ValueError."""
    if scaling is not None:
        unknown = sorted(k for k, v in scaling.items() if v is not None and k not in _SCALING_KEYS)
        if unknown:
            raise ValueError(f"rope scaling: {', '.join(map(str, unknown))} not served")
        own = scaling.get("rope_theta")
        if own is not None and theta is not None and float(own) != float(theta):
            raise ValueError(f"theta {theta} given, rope_theta {own} in the scaling")
        theta = own if theta is None else theta
    theta = 10000.0 if theta is None else theta
    f = float(theta) ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    kind = "default" if scaling is None else scaling.get("rope_type", scaling.get("type", "default"))
    if kind == "default":
        return f, 1.0
    if kind not in ("linear", "llama3", "yarn"):
        raise ValueError(f"rope scaling {kind!r} is not served")
    factor = float(scaling["factor"])
    if factor <= 0:
        raise ValueError(f"rope scaling factor {factor} must be positive")
    if kind == "linear":
        return f / factor, 1.0
    old = float(scaling["original_max_position_embeddings"])
    if kind == "llama3":
        lo, hi = float(scaling["low_freq_factor"]), float(scaling["high_freq_factor"])
        if not hi > lo:
            raise ValueError("rope scaling: high_freq_factor must exceed low_freq_factor")
        keep = ((old * f / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor, 1.0
    pair = lambda turns: dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = pair(float(scaling.get("beta_fast") or 32.0)), pair(float(scaling.get("beta_slow") or 1.0))
    if scaling.get("truncate") is None or scaling["truncate"]:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, dim - 1)
    ramp = ((torch.arange(dim // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
    m = scaling.get("attention_factor")
    if m is None:
        grow = lambda s: 0.1 * s * math.log(factor) + 1.0 if factor > 1.0 else 1.0  # noqa: E731
        one, every = scaling.get("mscale"), scaling.get("mscale_all_dim")
        m = grow(float(one)) / grow(float(every)) if one and every else grow(1.0)
    return f * (1.0 - ramp) + f / factor * ramp, float(m)


class _Rotate(torch.autograd.Function):
    """q, k turned; the gradient of a turn is the turn the other way, its
    tangent the tangent turned."""

    @staticmethod
    def forward(ctx, q, k, positions, rotary, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions)
        ctx.save_for_forward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        return rotary._launch(q, k, positions, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        (positions,) = ctx.saved_tensors
        rot, inv = ctx.rotary, not ctx.inverse
        if gq is None and gk is None:
            return None, None, None, None, None
        if gq is None:
            gk, _ = _turned(gk, None, positions, rot, inv)
        else:
            gq, gk = _turned(gq, gk, positions, rot, inv)
        return gq, gk, None, None, None

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return _turned(tq, tk, *ctx.saved_tensors, ctx.rotary, ctx.inverse)


def _turned(q, k, positions, rotary, inverse):
    """q and k (or None) turned, each as a function of its input if something
    is to be derived through that, else as a constant."""
    want = [_wants(t) for t in (q, k) if t is not None]
    if not any(map(any, want)):
        return rotary._launch(q, k, positions, inverse)
    if want[0] == want[-1]:
        return _Rotate.apply(q, k, positions, rotary, inverse)
    return tuple(_turned(t, None, positions, rotary, inverse)[0] for t in (q, k))


class Rotary:
    """Rotary positions: the first ``dim`` values of a head turn in pairs.

    Pair i turns by ``position * frequency[i]`` (``rope_frequencies``); pairs
    are (i, i + dim / 2) for ``layout="half"``, (2i, 2i + 1) for
    ``"interleaved"``.  Angles, their cosines and sines are computed once in
    float64 for positions below ``max_pos`` and kept as float32 tables (the
    attention factor multiplied in)."""

    def __init__(self, dim, max_pos, theta=None, layout="half", scaling=None, device="cuda"):
        if dim < 2 or dim % 2:
            raise ValueError(f"the rotated dim must be even and positive, got {dim}")
        if max_pos < 1:
            raise ValueError(f"max_pos must be positive, got {max_pos}")
        if layout not in ("half", "interleaved"):
            raise ValueError(f"layout must be 'half' or 'interleaved', got {layout!r}")
        self.dim, self.max_pos, self.layout = int(dim), int(max_pos), layout
        f, m = rope_frequencies(dim, theta, scaling)
        f = f.to(device)
        self.cos = torch.empty(self.max_pos, dim // 2, dtype=torch.float32, device=device)
        self.sin = torch.empty_like(self.cos)
        for i in range(0, self.max_pos, 65536):      # bounds the float64 temporaries
            t = torch.arange(i, min(i + 65536, self.max_pos), dtype=torch.float64, device=device)[:, None] * f
            self.cos[i:i + 65536], self.sin[i:i + 65536] = t.cos() * m, t.sin() * m

    def _rotation(self):
        return _abi.Rotation(self.cos.data_ptr(), self.sin.data_ptr(), self.max_pos, self.dim,
                             int(self.layout == "interleaved"))

    def rotate(self, q, k, positions):
        """q and k ([B, S, heads, D], one type) turned by their tokens'
        positions (broadcast to [B, S]).  Differentiable in both, in reverse
        and in forward mode; the output of one that needs no gradient needs
        none either."""
        if k is None:
            raise TypeError("rotate turns two tensors; call the rotation on one")
        call = _native()
        if call is not None:
            r = call.rotate(q, k, positions, self.cos, self.sin, self.layout == "interleaved")
            if r is not NotImplemented:
                return r
        self._check(q, k, positions)
        return _turned(q, k, positions, self, False)

    def __call__(self, x, positions):
        """One tensor [B, S, heads, D] turned."""
        call = _native()
        if call is not None:
            r = call.rotate(x, None, positions, self.cos, self.sin, self.layout == "interleaved")
            if r is not NotImplemented:
                return r
        self._check(x, None, positions)
        return _turned(x, None, positions, self, False)[0]

    def _check(self, q, k, positions):
        for t in (q, positions) if k is None else (q, k, positions):
            if not isinstance(t, torch.Tensor):
                raise TypeError(f"expected tensors, got {type(t).__name__}")
        _require(q, positions, self.cos, *(() if k is None else (k,)))
        if q.dim() != 4 or q.shape[-1] < self.dim:
            raise ValueError(f"expected [B, S, heads, D] with D >= {self.dim}, got {tuple(q.shape)}")
        if k is not None:
            if k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
                raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} differ in B, S or D")
            if k.dtype != q.dtype:
                raise TypeError(f"q is {q.dtype}, k {k.dtype}")

    def _launch(self, q, k, positions, inverse):
        q = _heads4("q", q)
        qo, ko = torch.empty(q.shape, dtype=q.dtype, device=q.device), None
        kh = None
        if k is not None:
            k = _heads4("k", k)
            ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            kh = ctypes.byref(_heads(k)) if k.shape[2] else None
        if q.numel() == 0 and (k is None or k.numel() == 0):
            return qo, ko
        tok, _keep = _tokens(q.shape[:2], positions)
        # a first tensor always has heads; k takes q's place where only it has
        xh, xo, yh, yo = (_heads(q), qo, kh, ko) if q.shape[2] else (_heads(k), ko, None, None)
        _run("ep_rotate", _abi.lib.ep_rotate(
            xh, yh, self._rotation(), tok, q.shape[3], int(inverse), xo.data_ptr(),
            yo.data_ptr() if yo is not None else None, _abi.stream_handle(q.device)))
        return qo, ko


class PagedKVCache:
    """One layer's keys and values in pages that sequences own by table.

    ``k`` and ``v`` are ``[n_pages, heads, page, D]`` in ``dtype``: bfloat16,
    float16, float8_e4m3fn or int8.  An 8-bit row (one head's values of one
    position) stands for code * scale, its scale in ``k_scale`` / ``v_scale``
    ``[n_pages, heads, page]`` (float32).  ``page`` is a power of two from 16
    to 1024, D a multiple of 16 up to 256.  Nothing is derived through a
    cache: a call that would have to raises."""

    def __init__(self, n_pages, page, heads, dim, dtype=torch.bfloat16, device="cuda"):
        if dtype not in _abi.CACHE_DT:
            raise TypeError(f"cache type {dtype} is not served: {[str(d) for d in _abi.CACHE_DT]}")
        shape = (n_pages, heads, page, dim)
        # zeros through uint8: float8 tensors have few operators
        new = lambda: torch.zeros(n_pages, heads, page, dim * dtype.itemsize, dtype=torch.uint8,  # noqa: E731
                                  device=device).view(dtype)
        scales = [torch.ones(shape[:3], dtype=torch.float32, device=device) if dtype.itemsize == 1 else None
                  for _ in range(2)]
        self._take(new(), new(), *scales)

    @classmethod
    def of(cls, k, v, k_scale=None, v_scale=None):
        """A cache over tensors that exist (shared, not copied)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, k_scale, v_scale):
        if k.dtype not in _abi.CACHE_DT:
            raise TypeError(f"cache type {k.dtype} is not served: {[str(d) for d in _abi.CACHE_DT]}")
        if k.dim() != 4 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
            raise ValueError("k and v must be alike, [n_pages, heads, page, D]")
        n, h, page, d = k.shape
        if n < 1 or h < 1:
            raise ValueError("a cache has at least one page and one head")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"page of {page} rows: a power of two from 16 to 1024 is served")
        if d < 16 or d > 256 or d % 16:
            raise ValueError(f"heads of {d} values: multiples of 16 up to 256 are served")
        scaled = k.dtype.itemsize == 1
        for s in (k_scale, v_scale):
            if (s is not None) != scaled:
                raise ValueError("8-bit caches have scales, 16-bit ones none")
            if scaled and (s.shape != k.shape[:3] or s.dtype != torch.float32 or s.device != k.device):
                raise ValueError("scales must be float32 [n_pages, heads, page] on the cache's device")
        for t in (k, v, k_scale, v_scale):
            if t is not None and (not t.is_contiguous() or t.data_ptr() % 16):
                raise ValueError("cache tensors must be contiguous and 16-byte aligned")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.heads, self.page, self.dim, self.dtype = n, h, page, d, k.dtype

    def _held(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def _cache(self):
        ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        return _abi.KVCache(self.k.data_ptr(), self.v.data_ptr(), ptr(self.k_scale), ptr(self.v_scale),
                            _abi.CACHE_DT[self.dtype], self.heads, self.page, self.dim, self.n_pages)

    def append(self, k, v, positions, table, q=None, rotary=None):
        """Store the tokens' k and v ([B, S, heads, D]) at their positions.

        With ``rotary``, k is turned on its way into the cache and q (if
        given, [B, S, q heads, D]) on its way out; returns q turned, or None
        without q.  A turned key is rounded once, to the cache's type.  Tokens
        of one call at the same place of a page race: what it holds then is
        neither's for certain."""
        call = _native()
        if call is not None:
            cos, sin, inter = (None, None, False) if rotary is None else \
                (rotary.cos, rotary.sin, rotary.layout == "interleaved")
            r = call.append(k, v, positions, table, q, cos, sin, inter, self.k, self.v, self.k_scale, self.v_scale)
            if r is not NotImplemented:
                return r
        _no_grad(q, k, v, *self._held())
        _require(self.k, k, v, positions, table, *(() if q is None else (q,)),
                 *(() if rotary is None else (rotary.cos,)))
        k, v = _heads4("k", k), _heads4("v", v)
        if k.shape != v.shape or k.shape[2:] != (self.heads, self.dim):
            raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} must be [B, S, {self.heads}, {self.dim}]")
        if k.dtype != v.dtype or (q is not None and q.dtype != k.dtype):
            raise TypeError("q, k and v must have one type")
        if rotary is not None and rotary.dim > self.dim:
            raise ValueError(f"a rotation of {rotary.dim} values in heads of {self.dim}")
        qo = None
        if q is not None:
            q = _heads4("q", q)
            if q.shape[:2] != k.shape[:2] or q.shape[3] != self.dim:
                raise ValueError(f"q must be [B, S, heads, {self.dim}] with k's B and S, got {tuple(q.shape)}")
            qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        tok, _keep = _tokens(k.shape[:2], positions, table)
        if k.numel() == 0:
            return qo
        some_q = q is not None and q.shape[2] > 0
        _run("ep_kv_append", _abi.lib.ep_kv_append(
            _heads(q) if some_q else None, _heads(k), _heads(v), rotary._rotation() if rotary is not None else None,
            tok, self._cache(), qo.data_ptr() if some_q else None, _abi.stream_handle(k.device)))
        return qo

    def read(self, positions, table, dtype=torch.bfloat16):
        """(k, v) [B, S, heads, D] in ``dtype``: the rows at positions [B, S]."""
        call = _native()
        if call is not None:
            r = call.read(positions, table, dtype, self.k, self.v, self.k_scale, self.v_scale)
            if r is not NotImplemented:
                return r
        _no_grad(*self._held())
        _require(self.k, positions, table)
        if _abi.dtype_code(dtype) is None:
            raise TypeError(f"the cache is read as float32, float16 or bfloat16, not {dtype}")
        if positions.dim() != 2:
            raise ValueError(f"positions must be [B, S], got {tuple(positions.shape)}")
        tok, _keep = _tokens(positions.shape, positions, table)
        shape = (*positions.shape, self.heads, self.dim)
        k = torch.empty(shape, dtype=dtype, device=self.k.device)
        v = torch.empty_like(k)
        if k.numel():
            _run("ep_kv_read", _abi.lib.ep_kv_read(tok, self._cache(), k.data_ptr(), v.data_ptr(),
                                                   _abi.dtype_code(dtype), _abi.stream_handle(k.device)))
        return k, v

    def attend(self, q, positions, table, scale=None, window=None):
        """Attention of q's tokens ([B, S, q heads, D], float16 or bfloat16)
        over positions ``max(0, p - window + 1) .. p`` of their sequences, p
        their own position (append them first); [B, S, q heads, D] in q's
        type.  ``scale`` defaults to D ** -0.5, ``window`` to all.  A 16-bit
        cache must have q's type.  Meant for one new token, or a few."""
        call = _native()
        if call is not None:
            r = call.attend(q, positions, table, scale, window, self.k, self.v, self.k_scale, self.v_scale)
            if r is not NotImplemented:
                return r
        _no_grad(q, *self._held())
        _require(self.k, q, positions, table)
        q = _heads4("q", q)
        if q.shape[3] != self.dim or q.shape[2] == 0 or q.shape[2] % self.heads:
            raise ValueError(f"q must be [B, S, n * {self.heads}, {self.dim}], got {tuple(q.shape)}")
        if q.dtype == torch.float32:
            raise TypeError("attention takes float16 or bfloat16 queries")
        if self.dtype.itemsize == 2 and q.dtype != self.dtype:
            raise TypeError(f"q is {q.dtype} over a cache of {self.dtype}")
        if window is not None and window < 1:
            raise ValueError(f"window must be positive, got {window}")
        if q.data_ptr() % 16 or any(n > 1 and s % 8 for n, s in zip(q.shape[:3], q.stride()[:3])):
            q = q.contiguous() if not q.is_contiguous() else q.clone()
        tok, _keep = _tokens(q.shape[:2], positions, table)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        if q.numel() == 0:
            return out
        qh, cache = _heads(q), self._cache()
        n = _abi.lib.ep_paged_attention_workspace(qh, tok, cache)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        _run("ep_paged_attention", _abi.lib.ep_paged_attention(
            qh, tok, cache, self.dim ** -0.5 if scale is None else float(scale),
            min(int(window or 0), 2 ** 63 - 1), out.data_ptr(),     # 64 bits there: more would wrap
            ws.data_ptr() if n else None, n, _abi.stream_handle(q.device)))
        return out

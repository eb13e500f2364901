"""Plain restatements of the paged operators (include/epure_paged.h) on the
CPU, from their definitions: rotary positions and attention in float64, the
cache's 8-bit rows in float32, where each step of the definition rounds.

Pinned by tests/test_paged_cpu.py (rotations as complex products, codes by
brute force over the representable values, attention against a softmax over
an explicit list of positions)."""
import math

import torch


def rotate(x, positions, cos, sin, interleaved=False, inverse=False):
    """float64 [B, S, heads, D] turned; cos / sin [max_pos, dim / 2].  A negative
    position gives zeros, one past the tables NaN."""
    x = x.detach().cpu().double()
    cos, sin = cos.detach().cpu().double(), sin.detach().cpu().double()
    if inverse:
        sin = -sin
    pos = positions.cpu().expand(x.shape[:2])
    half = cos.shape[1]
    ok = (pos >= 0) & (pos < cos.shape[0])
    at = torch.where(ok, pos, 0)
    c, s = cos[at][:, :, None, :], sin[at][:, :, None, :]
    y = x.clone()
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    y[(pos < 0)] = 0.0
    y[(pos >= cos.shape[0])] = math.nan
    return y


def rotate32(x, positions, cos, sin, interleaved=False):
    """The same in float32 steps (product, product, sum), for bit-exact checks."""
    x = x.detach().cpu().float()
    c, s = cos.cpu()[positions.cpu()][:, :, None, :], sin.cpu()[positions.cpu()][:, :, None, :]
    half = cos.shape[1]
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    y = x.clone()
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def held(x, dtype):
    """(codes as float32, scale [..., 1]) of f32 rows x in an 8-bit cache; (x in dtype, None) in a 16-bit one."""
    x = x.detach().cpu().float()
    if dtype.itemsize == 2:
        return x.to(dtype).float(), None
    m = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(m)
    safe = torch.where(bad, torch.ones_like(m), m)
    if dtype == torch.int8:
        top = safe.clamp(min=2.0 ** -100)
        n = torch.full_like(top, 127.0)
        scale = top / n
        codes = (x * (n / top)).round().clamp(-127, 127)
    else:
        scale = torch.empty_like(safe)
        for i, v in enumerate(safe.flatten().tolist()):
            e = -100
            while v > 448.0 * 2.0 ** e:
                e += 1
            scale.view(-1)[i] = 2.0 ** e
        codes = (x / scale).to(dtype).float()
    return torch.where(bad, torch.zeros_like(codes), codes), torch.where(bad, torch.full_like(scale, math.nan), scale)


def stands_for(x, dtype):
    """float32 values that the cache holds for f32 rows x."""
    codes, scale = held(x, dtype)
    return codes if scale is None else codes * scale


def attend(q, k, v, positions, scale, window=None):
    """float64 attention over contexts k, v [B, L, heads, D] (position j in
    row j): (output, sum of weight * |v|, largest sum of |q k| times scale)
    per query row.  Only positions that a row attends to are touched."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, S, H, D = q.shape
    G = H // k.shape[2]
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    big = torch.zeros(B, S, H, 1, dtype=torch.float64)
    for b in range(B):
        for s in range(S):
            p = int(positions[b, s])
            if p < 0:
                continue
            if p >= k.shape[1]:
                out[b, s] = math.nan
                continue
            lo = max(0, p - window + 1) if window else 0
            for h in range(H):
                kk, vv = k[b, lo:p + 1, h // G], v[b, lo:p + 1, h // G]
                sc = kk @ q[b, s, h] * scale
                w = torch.softmax(sc, 0)
                out[b, s, h], mag[b, s, h] = w @ vv, w @ vv.abs()
                big[b, s, h] = (kk.abs() @ q[b, s, h].abs()).max() * abs(scale)
    return out, mag, big


def half_step(x, dtype):
    """Half a step of ``dtype`` at x: relative, and below the normal numbers
    (f16: 2^-14) half the spacing there."""
    f = torch.finfo(dtype)
    return torch.clamp(f.eps / 2 * x.abs(), min=f.eps * f.smallest_normal / 2)


def attend_tolerance(out, mag, big, dtype, D):
    """Bound on |kernel - oracle|.  The output's rounding: half a step
    (``half_step``).  A score's f32 sum of D products and its scaling: (D + 4) 2^-24 of the sum
    of magnitudes; it moves a weight by that much relatively, and the weights'
    sum as well.  The rest relative to sum w |v|: weights enter their product
    as two 16-bit terms (2^-16), the exponential and the f32 sums over up to
    some thousand positions in blocks (2^-16 each): 2^-14 covers them."""
    delta = (D + 4) * 2.0 ** -24 * big
    return half_step(out, dtype) + (2.0 ** -14 + 2 * delta) * mag

"""The operators between a served decoder's packed linears, as cases that can
be timed: rotary positions, a paged key-value cache that is quantised as it
is written, and attention of new tokens over it.

Four kinds of call:

* ``rotate``: ``Rotary.rotate(q, k, positions)``; with ``grad`` also the
  gradients of q and k (a training step's share of it);
* ``append``: ``PagedKVCache.append`` of new tokens' keys and values, q and k
  rotated on the way.  An 8-bit cache is read back where it was written, so
  that the outputs are the values it stands for; a 16-bit cache is returned;
* ``read``: ``PagedKVCache.read`` of whole contexts;
* ``attend``: ``PagedKVCache.attend`` of each sequence's newest token (or the
  newest few) over its context.

Definitions.  A pair (a, b) of a head turns by t = position * frequency:
(a cos t - b sin t, b cos t + a sin t), times the attention factor of the
frequencies' scaling.  A cache row of 8 bits holds codes c and a scale s:
int8: s = max|x| / 127, c = rint(x * (127 / max|x|)); e4m3: s = 2^e with the
least e for which max|x| <= 448 * 2^e, c = x / s rounded to e4m3; it stands
for c * s.  A token at position p sees positions p - window + 1 .. p.

Head counts and sizes are those of the decoder list in ``epure.decode`` or
generic.  Queries, keys and values are normal; queries are twice as wide, so
that the softmax is neither flat nor one position.
"""
import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LLAMA3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
LINEAR = {"rope_type": "linear", "factor": 2.0}
SCALINGS = {"none": None, "linear": LINEAR, "llama3": LLAMA3, "yarn": YARN}


# ------------------------------------------------------------------ the cases
def _rotate(name, batch, seq, start, heads, kv, dim, rot, layout, scaling, dtype, grad=False):
    return {"name": name, "kind": "rotate", "batch": batch, "seq": seq, "start": start, "heads": heads, "kv": kv,
            "dim": dim, "rot": rot, "layout": layout, "scaling": scaling, "dtype": dtype, "grad": grad}


def _append(name, batch, new, lo, hi, heads, kv, dim, page, cache, dtype):
    return {"name": name, "kind": "append", "batch": batch, "new": new, "lo": lo, "hi": hi, "heads": heads,
            "kv": kv, "dim": dim, "page": page, "cache": cache, "dtype": dtype}


def _read(name, batch, lo, hi, kv, dim, page, cache, dtype):
    return {"name": name, "kind": "read", "batch": batch, "lo": lo, "hi": hi, "kv": kv, "dim": dim, "page": page,
            "cache": cache, "dtype": dtype}


def _attend(name, batch, new, lo, hi, heads, kv, dim, page, cache, dtype, window=0):
    return {"name": name, "kind": "attend", "batch": batch, "new": new, "lo": lo, "hi": hi, "heads": heads,
            "kv": kv, "dim": dim, "page": page, "cache": cache, "dtype": dtype, "window": window}


def listed():
    return [
        # one decoded token of one sequence (Qwen3-1.7B heads): latency
        _rotate("rotate_token", 1, 1, 777, 16, 8, 128, 128, "half", "none", "bf16"),
        # four prompts of 4096 tokens far into a long context (Llama-3-8B heads)
        _rotate("rotate_prompt_4x4096", 4, 4096, 100000, 32, 8, 128, 128, "half", "llama3", "bf16"),
        # a training step over ragged sizes: part of the head, interleaved pairs, forward and gradients
        _rotate("rotate_train_3x1021", 3, 1021, 0, 20, 4, 96, 64, "interleaved", "yarn", "f16", True),
        # a decode step's writes: one token each of 64 sequences into an int8 cache
        _append("append_64x1_int8", 64, 1, 100, 4000, 32, 8, 128, 64, "int8", "bf16"),
        # two prompts of up to 4096 tokens into an e4m3 cache
        _append("append_2x4096_e4m3", 2, 4096, 3001, 4096, 32, 8, 128, 128, "e4m3", "bf16"),
        # a small decode batch into a 16-bit cache of small pages
        _append("append_8x1_bf16", 8, 1, 17, 301, 16, 8, 128, 16, "bf16", "bf16"),
        # eight contexts read back out of an int8 cache (a prefix handed on, a cache moved)
        _read("read_8x4096_int8", 8, 1000, 4096, 8, 128, 64, "int8", "bf16"),
        # one short sequence (Qwen3-1.7B heads): latency
        _attend("attend_1x129_bf16", 1, 1, 129, 129, 16, 8, 128, 16, "bf16", "bf16"),
        # an ordinary decode batch of ragged lengths (Llama-3-8B heads)
        _attend("attend_32x4096_bf16", 32, 1, 1, 4096, 32, 8, 128, 64, "bf16", "bf16"),
        # the same from an int8 cache: more and longer sequences in the same memory
        _attend("attend_48x8192_int8", 48, 1, 500, 8192, 32, 8, 128, 32, "int8", "bf16"),
        # four sequences of long contexts: the largest
        _attend("attend_4x131072_bf16", 4, 1, 120000, 131072, 32, 8, 128, 128, "bf16", "bf16"),
        # five tokens at once (drafted tokens being verified) with a sliding window, five query heads to a
        # key head, an e4m3 cache
        _attend("attend_8x5_e4m3_window", 8, 5, 3, 6001, 20, 4, 80, 16, "e4m3", "f16", 1500),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv


def draw(rng):
    """One more call of the same ranges: 1 to 64 sequences, 1 to 131072
    positions, one to eight new tokens (or prompts), heads of 64 to 256
    values in 1 to 8 key heads, pages of 16 to 256 rows."""
    kind = rng.choice(["rotate", "append", "read", "attend", "attend"])
    heads, kv = _heads(rng)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    cache = rng.choice(["bf16", "f16", "int8", "e4m3"])
    dtype = cache if cache in ("bf16", "f16") else rng.choice(["bf16", "f16"])
    if kind == "rotate":
        batch, seq = _log(rng, 1, 8), _log(rng, 1, 4096)
        rot = rng.choice([dim, dim, dim // 2, 32])
        c = _rotate("", batch, seq, rng.choice([0, _log(rng, 1, 120000)]), heads, kv, dim, rot,
                    rng.choice(["half", "interleaved"]), rng.choice(list(SCALINGS)),
                    rng.choice(["f32", "f16", "bf16"]), rng.random() < 0.5)
        while _tokens(c) * (heads + kv) * dim > 4 * 4096 * 40 * 128:
            c["seq"] = c["seq"] // 2
    elif kind == "append":
        if rng.random() < 0.5:
            hi = _log(rng, 1, 16384)
            c = _append("", _log(rng, 1, 64), 1, _log(rng, 1, hi), hi, heads, kv, dim, page, cache, dtype)
        else:
            hi = _log(rng, 2, 4096)
            c = _append("", _log(rng, 1, 8), hi, _log(rng, 1, hi), hi, heads, kv, dim, page, cache, dtype)
        while c["batch"] > 1 and (c["batch"] * hi * kv * dim > 1 << 26 or c["batch"] * c["new"] * heads * dim > 1 << 26):
            c["batch"] //= 2
    elif kind == "read":
        hi = _log(rng, 1, 8192)
        c = _read("", _log(rng, 1, 16), _log(rng, 1, hi), hi, kv, dim, page, cache, dtype)
        while c["batch"] > 1 and c["batch"] * hi * kv * dim > 1 << 26:
            c["batch"] //= 2
    else:
        hi = _log(rng, 1, 131072)
        c = _attend("", _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 3, 5, 8]), _log(rng, 1, hi), hi, heads, kv, dim,
                    page, cache, dtype, rng.choice([0, 0, 0, _log(rng, 1, 8192)]))
        # the plain form widens the padded contexts and scores to 32 bits: no more of them than in the largest listed case
        while c["batch"] > 1 and (c["batch"] * hi * kv * dim > 4 * 131072 * 8 * 128
                                  or c["batch"] * hi * heads * c["new"] > 4 * 131072 * 32 * 4):
            c["batch"] //= 2
    del c["name"]
    return c


def _tokens(c):
    return c["batch"] * c["seq"]


def _lengths(c):
    """Context lengths of the sequences, spread evenly from lo to hi."""
    lo, hi, n = min(c["lo"], c["hi"]), c["hi"], c["batch"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _seen(c):
    """Cache positions that an ``attend`` call reads, over all sequences."""
    total = 0
    for n in _lengths(c):
        first = max(n - c["new"], 0)
        total += n - (max(first - c["window"] + 1, 0) if c["window"] else 0)
    return total


def _pairs(c):
    """(new token, position) pairs that an ``attend`` call scores."""
    total = 0
    for n in _lengths(c):
        for p in range(max(n - c["new"], 0), n):
            total += min(p + 1, c["window"]) if c["window"] else p + 1
    return total


def _size(name):
    return TYPES[name].itemsize


def _row(c):
    """Bytes of one cache row of one head."""
    return c["dim"] * _size(c["cache"]) + (4 if _size(c["cache"]) == 1 else 0)


def work(c):
    if c["kind"] == "rotate":
        values = _tokens(c) * (c["heads"] + c["kv"]) * c["dim"]
        once = 2 * values * _size(c["dtype"]) + _tokens(c) * 8 + c["seq"] * c["rot"] * 4
        n = 2 if c["grad"] else 1
        return {"bytes": n * once, "flops": n * 3 * values * c["rot"] // c["dim"]}
    lengths = _lengths(c)
    tables = 4 * sum((n + c["page"] - 1) // c["page"] for n in lengths)
    if c["kind"] == "append":
        tokens = sum(lengths) if c["new"] > 1 else c["batch"]
        q, k = tokens * c["heads"] * c["dim"], tokens * c["kv"] * c["dim"]
        rows = 2 * tokens * c["kv"] * _row(c)
        b = 2 * q * _size(c["dtype"]) + 2 * k * _size(c["dtype"]) + rows + tokens * (8 + 4 * c["dim"]) + tables
        if _size(c["cache"]) == 1:
            b += rows + 2 * k * _size(c["dtype"])       # read back
        return {"bytes": b, "flops": 3 * (q + k) + 4 * k}
    if c["kind"] == "read":
        rows = 2 * sum(lengths) * c["kv"]
        return {"bytes": rows * (_row(c) + c["dim"] * _size(c["dtype"])) + sum(lengths) * 8 + tables,
                "flops": rows * c["dim"]}
    q = c["batch"] * c["new"] * c["heads"] * c["dim"] * _size(c["dtype"])
    return {"bytes": 2 * _seen(c) * c["kv"] * _row(c) + 2 * q + c["batch"] * c["new"] * 8 + tables,
            "flops": 4 * c["heads"] * c["dim"] * _pairs(c)}


# ------------------------------------------------------------------ inputs
def _frequencies(rot, theta, scaling):
    """Angles per position of the rot / 2 pairs (f64) and the attention factor."""
    f = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling is None:
        return f, 1.0
    kind, factor = scaling["rope_type"], scaling["factor"]
    if kind == "linear":
        return f / factor, 1.0
    old = scaling["original_max_position_embeddings"]
    if kind == "llama3":
        lo, hi = scaling["low_freq_factor"], scaling["high_freq_factor"]
        turns = old * f / (2 * math.pi)                       # turns within the original context
        keep = ((turns - lo) / (hi - lo)).clamp(0, 1)
        return keep * f + (1 - keep) * f / factor, 1.0
    at = lambda turns: rot * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * (1 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)


def _power(e):
    """2^e as f32, from its bits."""
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x, cache):
    """Codes and row scales of f32 rows x."""
    amax = x.abs().amax(-1, keepdim=True)
    if cache == "int8":
        m = amax.clamp(min=2.0 ** -100)
        n = torch.full_like(m, 127.0)
        s = torch.div(m, n)
        c = (x * torch.div(n, m)).round().clamp(-127, 127).to(torch.int8)
    else:
        frac, e = torch.frexp(amax)
        e = torch.where(frac <= 0.875, e - 9, e - 8).clamp(min=-100)
        s = _power(e)
        c = (x * _power(-e)).to(torch.float8_e4m3fn)
    ok = torch.isfinite(amax)
    return c, torch.where(ok, s, float("nan")).squeeze(-1)


def _pool(c, g, pages, filled):
    """Cache tensors of ``pages`` pages: k, v, k_scale, v_scale."""
    shape = (pages, c["kv"], c["page"], c["dim"])
    dt = TYPES[c["cache"]]
    out = [torch.zeros(shape, dtype=torch.uint8, device=DEV).view(dt) if dt.itemsize == 1
           else torch.zeros(shape, dtype=dt, device=DEV) for _ in range(2)]
    scales = [torch.ones(shape[:3], device=DEV) if dt.itemsize == 1 else None for _ in range(2)]
    if filled:
        step = max(1, (1 << 26) // (c["kv"] * c["page"] * c["dim"]))
        for t, s in zip(out, scales):
            for i in range(0, pages, step):
                x = torch.randn((min(step, pages - i),) + shape[1:], generator=g, device=DEV)
                if s is None:
                    t[i:i + step] = x.to(dt)
                else:
                    t[i:i + step], s[i:i + step] = _quantise(x, c["cache"])
    return out + scales


def prepare(c, seed):
    g = _gen(seed)
    st = {"case": c}
    if c["kind"] == "rotate":
        shape = (c["batch"], c["seq"])
        dt = TYPES[c["dtype"]]
        st["q"] = _normal(g, shape + (c["heads"], c["dim"]), dt).requires_grad_(c["grad"])
        st["k"] = _normal(g, shape + (c["kv"], c["dim"]), dt).requires_grad_(c["grad"])
        if c["grad"]:
            st["gq"], st["gk"] = _normal(g, st["q"].shape, dt, 0.01), _normal(g, st["k"].shape, dt, 0.01)
        st["positions"] = (c["start"] + torch.arange(c["seq"], device=DEV)).expand(shape).contiguous()
        st["max_pos"] = c["start"] + c["seq"]
        _keep_rotary(st, c["rot"], c["layout"], SCALINGS[c["scaling"]])
        return st
    lengths = _lengths(c)
    need = [(n + c["page"] - 1) // c["page"] for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["batch"], max(need)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    st["table"] = table
    st["pool"] = _pool(c, g, pages, c["kind"] != "append")
    ends = torch.tensor(lengths, device=DEV)
    if c["kind"] == "read" or (c["kind"] == "append" and c["new"] > 1):
        p = torch.arange(max(lengths), device=DEV).expand(c["batch"], -1)
        st["positions"] = torch.where(p < ends[:, None], p, -1)      # shorter sequences are padded
    else:
        new = c["new"]
        p = ends[:, None] - new + torch.arange(new, device=DEV)
        st["positions"] = p.clamp(min=-1)
    shape = tuple(st["positions"].shape)
    dt = TYPES[c["dtype"]]
    if c["kind"] in ("append", "attend"):
        st["q"] = _normal(g, shape + (c["heads"], c["dim"]), dt, 2.0)
    if c["kind"] == "append":
        # keys and values as a projection gives them: one row of q|k|v a token
        kv = _normal(g, shape + (2 * c["kv"], c["dim"]), dt)
        st["k"], st["v"] = kv[..., :c["kv"], :], kv[..., c["kv"]:, :]
        st["max_pos"] = max(lengths)
        _keep_rotary(st, c["dim"], "half", None)
    if own:
        _handle(st)
    return st


def _keep_rotary(st, rot, layout, scaling):
    """What a program keeps for the rotation: the framework's handle, or cos / sin tables."""
    st["rot"], st["layout"], st["scaling"] = rot, layout, scaling
    if own:
        _rotary(st)
    else:
        _tables(st)


def _tables(st):
    if "cos" not in st:
        f, m = _frequencies(st["rot"], 5e5, st["scaling"])
        t = torch.arange(st["max_pos"], dtype=torch.float64, device=DEV)[:, None] * f.to(DEV)
        st["cos"], st["sin"] = (t.cos() * m).float(), (t.sin() * m).float()
    return st["cos"], st["sin"]


def _epure():
    path = os.path.join(_ROOT, "epure-runtime_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import epure
    return epure


def _rotary(st):
    if "rotary" not in st:
        st["rotary"] = _epure().Rotary(st["rot"], st["max_pos"], theta=5e5, layout=st["layout"],
                                       scaling=st["scaling"], device=DEV)
    return st["rotary"]


def _handle(st):
    if "cache" not in st:
        st["cache"] = _epure().PagedKVCache.of(*st["pool"])
    return st["cache"]


# ------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, rot, layout):
    """f32 x with its first ``rot`` values turned; cos, sin broadcast over [..., rot / 2]."""
    r = x[..., :rot]
    if layout == "half":
        a, b = r[..., :rot // 2], r[..., rot // 2:]
    else:
        a, b = r[..., 0::2], r[..., 1::2]
    ta, tb = a * cos - b * sin, b * cos + a * sin
    t = torch.cat((ta, tb), -1) if layout == "half" else torch.stack((ta, tb), -1).flatten(-2)
    return torch.cat((t, x[..., rot:]), -1)


def _rows(table, positions, page):
    """(page, row) of every position; padding (position -1) points at row 0 of some page."""
    p = positions.clamp(min=0)
    return table.long().gather(1, p // page).clamp(min=0), p % page


def _plain_rotate(st, q, k, gq=None, gk=None):
    cos, sin = (t[st["positions"]][:, :, None, :] for t in _tables(st))
    if gq is None:
        return [_turn(x.float(), cos, sin, st["rot"], st["layout"]).to(x.dtype) for x in (q, k)]
    return [_turn(x.float(), cos, -sin, st["rot"], st["layout"]).to(x.dtype) for x in (gq, gk)]


def _plain_append(c, st):
    pos, pool = st["positions"], st["pool"]
    real = (pos >= 0)[:, :, None, None]
    cos, sin = (t[pos.clamp(min=0)][:, :, None, :] for t in _tables(st))
    q = torch.where(real, _turn(st["q"].float(), cos, sin, c["dim"], "half"), 0.0).to(st["q"].dtype)
    k = _turn(st["k"].float(), cos, sin, c["dim"], "half")
    page, row = _rows(st["table"], pos, c["page"])
    at = pos >= 0
    real_rows = (lambda x: x[at]) if c["new"] > 1 else (lambda x: x.flatten(0, 1))   # one token: no padding
    pg, rw = real_rows(page), real_rows(row)
    if pool[2] is None:
        pool[0][pg, :, rw] = real_rows(k).to(pool[0].dtype)
        pool[1][pg, :, rw] = real_rows(st["v"]).to(pool[1].dtype)
        return [q, pool[0], pool[1]]
    for x, t, s in ((k, pool[0], pool[2]), (st["v"].float(), pool[1], pool[3])):
        codes, scale = _quantise(real_rows(x), c["cache"])
        t.view(torch.uint8)[pg, :, rw] = codes.view(torch.uint8)
        s[pg, :, rw] = scale
    return [q] + _plain_read(c, st)


def _plain_read(c, st):
    pos, pool = st["positions"], st["pool"]
    page, row = _rows(st["table"], pos, c["page"])
    out = []
    for t, s in zip(pool[:2], pool[2:]):
        x = t.view(torch.uint8)[page, :, row].view(t.dtype).float() if s is not None else t[page, :, row].float()
        if s is not None:
            x = x * s[page, :, row][..., None]
        out.append(torch.where((pos >= 0)[:, :, None, None], x, 0.0).to(TYPES[c["dtype"]]))
    return out


def _context(t, s, table):
    """All pages of every sequence in order, f32 [batch, kv, positions, dim]."""
    idx = table.long().clamp(min=0)
    x = t.view(torch.uint8)[idx].view(t.dtype).float() if s is not None else t[idx].float()
    if s is not None:
        x = x * s[idx][..., None]
    b, w, h, p, d = x.shape
    return x.transpose(1, 2).reshape(b, h, w * p, d)


def _plain_attend(c, st):
    q, pos, pool = st["q"], st["positions"], st["pool"]
    b, n, heads, d = q.shape
    kv, g = c["kv"], heads // c["kv"]
    k = _context(pool[0], pool[2], st["table"])
    qh = q.float().view(b, n, kv, g, d).transpose(1, 2).reshape(b, kv, n * g, d)
    s = torch.matmul(qh, k.transpose(-1, -2)) * d ** -0.5
    del k
    j = torch.arange(s.shape[-1], device=q.device)
    ok = j <= pos[..., None]
    if c["window"]:
        ok = ok & (j > pos[..., None] - c["window"])
    ok = ok[:, None, :, None, :].expand(b, kv, n, g, -1).reshape(s.shape)
    s = s.masked_fill(~ok, float("-inf"))
    e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min))
    v = _context(pool[1], pool[3], st["table"])
    total = e.sum(-1, keepdim=True)
    o = torch.matmul(e, v) / torch.where(total > 0, total, 1.0)
    return o.view(b, kv, n, g, d).transpose(1, 2).reshape(b, n, heads, d).to(q.dtype)


# ------------------------------------------------------------------ one pass
def run(st):
    c = st["case"]
    if c["kind"] == "rotate":
        q, k = st["q"], st["k"]
        if not own:
            out = _plain_rotate(st, q.detach(), k.detach())
            return out + _plain_rotate(st, q, k, st["gq"], st["gk"]) if c["grad"] else out
        out = list(_rotary(st).rotate(q, k, st["positions"]))
        if c["grad"]:
            grads = torch.autograd.grad(out, (q, k), (st["gq"], st["gk"]))
            return [t.detach() for t in out] + list(grads)
        return out
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}[c["kind"]](c, st)
    cache, pos, table = _handle(st), st["positions"], st["table"]
    if c["kind"] == "append":
        q = cache.append(st["k"], st["v"], pos, table, q=st["q"], rotary=_rotary(st))
        if st["pool"][2] is None:
            return [q, cache.k, cache.v]
        return [q] + list(cache.read(pos, table, TYPES[c["dtype"]]))
    if c["kind"] == "read":
        return list(cache.read(pos, table, TYPES[c["dtype"]]))
    return cache.attend(st["q"], pos, table, window=c["window"] or None)


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_turn(st, x, back=False):
    f, m = _frequencies(st["rot"], 5e5, st["scaling"])
    t = st["positions"].clamp(min=0).double()[..., None, None] * f.to(DEV)
    z = torch.polar(torch.full_like(t, m), -t if back else t)
    x = x.detach().double()
    r = x[..., :st["rot"]]
    half = st["rot"] // 2
    u = torch.complex(r[..., :half], r[..., half:]) if st["layout"] == "half" else \
        torch.view_as_complex(r.unflatten(-1, (half, 2)).contiguous())
    y = u * z
    y = torch.cat((y.real, y.imag), -1) if st["layout"] == "half" else torch.view_as_real(y).flatten(-2)
    return torch.cat((y, x[..., st["rot"]:]), -1)


def _exact_held(x, cache):
    """The values that 8 bits hold of f64 rows x."""
    m = x.abs().amax(-1, keepdim=True)
    if cache == "int8":
        return (x * 127 / m).round() * (m / 127)
    e = torch.ceil(torch.log2(m / 448))
    e = torch.where(m <= 448 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(m > 448 * torch.exp2(e), e + 1, e)
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # spacing of e4m3 at y
    return (y / step).round() * step * torch.exp2(e)


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] == "rotate":
        out = [_exact_turn(st, st["q"]), _exact_turn(st, st["k"])]
        return out + [_exact_turn(st, st["gq"], True), _exact_turn(st, st["gk"], True)] if c["grad"] else out
    pos, table, pool = st["positions"], st["table"].long(), st["pool"]
    at = pos >= 0
    if c["kind"] == "append":
        pad = at[..., None, None]
        q = torch.where(pad, _exact_turn(st, st["q"]), 0.0)
        k, v = _exact_turn(st, st["k"]), st["v"].double()
        if pool[2] is not None:
            return [q] + [torch.where(pad, _exact_held(x, c["cache"]), 0.0) for x in (k, v)]
        out = [q]
        for x, t in ((k, pool[0]), (v, pool[1])):
            t = t.double()
            for b in range(c["batch"]):
                p = pos[b][at[b]]
                t[table[b, p // c["page"]], :, p % c["page"]] = x[b][at[b]]
            out.append(t)
        return out
    if c["kind"] == "read":
        out = []
        for t, s in zip(pool[:2], pool[2:]):
            o = torch.zeros(tuple(pos.shape) + (c["kv"], c["dim"]), dtype=torch.float64, device=DEV)
            for b in range(c["batch"]):
                p = pos[b][at[b]]
                o[b][at[b]] = _exact_rows(t, s, table[b], p, c["page"])
            out.append(o)
        return out
    q = st["q"].double()
    g = c["heads"] // c["kv"]
    out = torch.zeros_like(q)
    for b, n in enumerate(_lengths(c)):
        p = torch.arange(n, device=DEV)
        k, v = (_exact_rows(t, s, table[b], p, c["page"]) for t, s in zip(pool[:2], pool[2:]))
        for i in range(c["new"]):
            last = n - c["new"] + i
            if last < 0:
                continue
            first = max(last - c["window"] + 1, 0) if c["window"] else 0
            for h in range(c["kv"]):
                s = k[first:last + 1, h] @ q[b, i, h * g:(h + 1) * g].T * c["dim"] ** -0.5
                out[b, i, h * g:(h + 1) * g] = torch.softmax(s, 0).T @ v[first:last + 1, h]
    return out


def _exact_rows(t, s, pages, p, page):
    """f64 rows of one sequence at positions p: [len(p), kv, dim]."""
    pg, rw = pages[p // page], p % page
    if s is None:
        return t[pg, :, rw].double()
    return t.view(torch.uint8)[pg, :, rw].view(t.dtype).double() * s[pg, :, rw].double()[..., None]

"""What a served batch needs where contexts are shared, long, or run ahead of
with drafted tokens, as cases that can be timed:

* ``shared``: ``PagedKVCache.attend(..., shared=n)``: attention of a batch
  whose tables begin with the same n pages (a system prompt, a document asked
  about many times), those pages computed once for all of it;
* ``bounds``: ``PagedKVCache.append`` into a cache that keeps each page's
  smallest and largest key values.  An 8-bit cache is read back where it was
  written; a 16-bit cache is returned, and the bounds in either case;
* ``select``: ``PagedKVCache.select`` of the n pages of a context that matter
  most to each token, by the bounds, and ``attend(..., blocks=...)`` over them;
* ``verify``: ``verify_draft`` of drafted tokens against the target's
  probabilities.

Definitions.  Attention: softmax over j of scale q . k_j, applied to v_j, over
the positions p - window + 1 .. p of a token at position p.  Bounds of a page
and cache head: the least and the largest of the keys that the cache holds in
rows 0 .. r, r the last row written.  Score of a page for a token and a cache
head whose query heads are q_g: sum over d of
hi_d * sum_g max(q_gd, 0) + lo_d * sum_g min(q_gd, 0): the group's scores of
no position in the page sum to more.  The token's own page is always taken,
then those of the largest scores, the lower page first where they are equal.
Verification: drafted token x at step i stands if u_i q_i(x) < p_i(x), p the
target's and q the draft's probabilities (q = 1 where none are given); the
first that does not is replaced by the first v whose running sum of
max(p_i - q_i, 0) exceeds u_n times the whole sum (of p_i, where that sum is
zero), and where all stand, one more token is drawn from the target likewise.

Head counts and sizes are those of the decoder list in ``epure.decode`` or
generic.  Queries, keys and values are normal; queries are twice as wide, so
that the softmax is neither flat nor one position, and the keys of a page
lean one way, so that pages differ.
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


# ------------------------------------------------------------------ the cases
def _shared(name, batch, new, prefix, lo, hi, heads, kv, dim, page, cache, dtype, window=0):
    """``prefix`` positions in common (whole pages), then lo .. hi of each sequence's own."""
    return {"name": name, "kind": "shared", "batch": batch, "new": new, "prefix": prefix, "lo": lo, "hi": hi,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "cache": cache, "dtype": dtype, "window": window}


def _bounds(name, batch, new, lo, hi, kv, dim, page, cache, dtype):
    """One token of each sequence (new 1) or whole prompts of lo .. hi tokens (new = hi)."""
    return {"name": name, "kind": "bounds", "batch": batch, "new": new, "lo": lo, "hi": hi, "kv": kv, "dim": dim,
            "page": page, "cache": cache, "dtype": dtype}


def _select(name, batch, new, lo, hi, take, heads, kv, dim, page, cache, dtype):
    return {"name": name, "kind": "select", "batch": batch, "new": new, "lo": lo, "hi": hi, "take": take,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "cache": cache, "dtype": dtype}


def _verify(name, batch, drafted, vocab, dtype, draft):
    return {"name": name, "kind": "verify", "batch": batch, "drafted": drafted, "vocab": vocab, "dtype": dtype,
            "draft": draft}


def listed():
    return [
        # four short conversations behind one system prompt (Qwen3-1.7B heads): latency
        _shared("shared_4x1024_bf16", 4, 1, 1024, 1, 130, 16, 8, 128, 16, "bf16", "bf16"),
        # an ordinary decode batch behind a long system prompt (Llama-3-8B heads)
        _shared("shared_32x8192_bf16", 32, 1, 8192, 5, 600, 32, 8, 128, 64, "bf16", "bf16"),
        # the same from an int8 cache, many more sequences
        _shared("shared_128x16384_int8", 128, 1, 16384, 1, 300, 32, 8, 128, 32, "int8", "bf16"),
        # a book asked about 64 times: the largest
        _shared("shared_64x65536_bf16", 64, 1, 65536, 100, 2000, 32, 8, 128, 128, "bf16", "bf16"),
        # drafted tokens of nine sequences at once with a sliding window that ends inside the prefix, five query
        # heads to a key head, an e4m3 cache
        _shared("shared_9x5x2992_e4m3_window", 9, 5, 2992, 3, 801, 20, 4, 80, 16, "e4m3", "f16", 2501),
        # a decode step's writes into a cache that keeps bounds: one token each of 64 sequences
        _bounds("bounds_64x1_int8", 64, 1, 100, 4000, 8, 128, 64, "int8", "bf16"),
        # two prompts of up to 4096 tokens
        _bounds("bounds_2x4096_bf16", 2, 4096, 3001, 4096, 8, 128, 64, "bf16", "bf16"),
        # one sequence that has few more pages than are taken (Qwen3-1.7B heads): latency
        _select("select_1x700_bf16", 1, 1, 700, 700, 32, 16, 8, 128, 16, "bf16", "bf16"),
        # eight sequences of very long contexts, 4096 positions of each attended to (Llama-3-8B heads)
        _select("select_8x131072_bf16", 8, 1, 100000, 131072, 64, 32, 8, 128, 64, "bf16", "bf16"),
        # three drafted tokens of ragged sequences, three query heads to a key head, an int8 cache
        _select("select_20x3x9001_int8", 20, 3, 2, 9001, 47, 12, 4, 96, 32, "int8", "f16"),
        # four drafted tokens of one sequence: latency
        _verify("verify_1x4x32000_f32", 1, 4, 32000, "f32", True),
        # seven drafted tokens of each of 64 sequences over the Llama-3 vocabulary
        _verify("verify_64x7x128256_f32", 64, 7, 128256, "f32", True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 3, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv


def draw(rng):
    """One more call of the same ranges: 1 to 128 sequences, up to 131072
    positions, one to eight new tokens (or prompts), heads of 64 to 256
    values in 1 to 8 key heads, pages of 16 to 256 rows, vocabularies of 1000
    to 160000."""
    kind = rng.choice(["shared", "shared", "bounds", "select", "select", "verify"])
    heads, kv = _heads(rng)
    dim = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    cache = rng.choice(["bf16", "f16", "int8", "e4m3"])
    dtype = cache if cache in ("bf16", "f16") else rng.choice(["bf16", "f16"])
    new = rng.choice([1, 1, 1, 2, 3, 5, 8])
    if kind == "shared":
        prefix = max(_log(rng, 16, 65536) // page, 1) * page
        hi = _log(rng, 1, 4096)
        c = _shared("", _log(rng, 1, 128), new, prefix, _log(rng, 1, hi), hi, heads, kv, dim, page, cache, dtype,
                    rng.choice([0, 0, 0, _log(rng, 1, 16384)]))
        # the plain form holds scores and contexts in 32 bits: no more of them than in the largest listed case
        while c["batch"] > 1 and (c["batch"] * new * heads * (prefix + hi) > 64 * 32 * 65536
                                  or c["batch"] * hi * kv * dim > 64 * 2000 * 8 * 128):
            c["batch"] //= 2
    elif kind == "bounds":
        if rng.random() < 0.5:
            hi = _log(rng, 1, 16384)
            c = _bounds("", _log(rng, 1, 64), 1, _log(rng, 1, hi), hi, kv, dim, page, cache, dtype)
        else:
            hi = _log(rng, 2, 4096)
            c = _bounds("", _log(rng, 1, 8), hi, _log(rng, 1, hi), hi, kv, dim, page, cache, dtype)
        while c["batch"] > 1 and c["batch"] * hi * kv * dim > 1 << 25:
            c["batch"] //= 2
    elif kind == "select":
        hi = _log(rng, 1, 131072)
        c = _select("", _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 3]), _log(rng, 1, hi), hi, _log(rng, 1, 128), heads,
                    kv, dim, page, cache, dtype)
        while c["batch"] > 1 and (c["batch"] * hi * kv * dim > 8 * 131072 * 8 * 128
                                  or c["batch"] * c["new"] * kv * c["take"] * page * dim > 1 << 27):
            c["batch"] //= 2
    else:
        c = _verify("", _log(rng, 1, 64), rng.randint(1, 8), _log(rng, 1000, 160000), rng.choice(["f32", "f16", "bf16"]),
                    rng.random() < 0.7)
        while c["batch"] * (2 * c["drafted"] + 1) * c["vocab"] > 64 * 15 * 128256:
            c["batch"] //= 2
    del c["name"]
    return c


def _lengths(c):
    """Lengths of the sequences (behind the shared pages), spread evenly from lo to hi."""
    lo, hi, n = min(c["lo"], c["hi"]), c["hi"], c["batch"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _size(name):
    return TYPES[name].itemsize


def _row(c):
    """Bytes of one cache row of one head."""
    return c["dim"] * _size(c["cache"]) + (4 if _size(c["cache"]) == 1 else 0)


def _bounds_row(c):
    """Bytes of the bounds of one page of one head."""
    return 2 * c["dim"] * (2 if _size(c["cache"]) == 2 else 4)


def work(c):
    if c["kind"] == "verify":
        n, k = c["batch"], 2 if c["draft"] else 1
        # whole rows of the step that ends it, two numbers of every step before
        return {"bytes": n * (k * c["vocab"] * _size(c["dtype"]) + c["drafted"] * (8 + 4 + 2 * _size(c["dtype"]) + 8)),
                "flops": 3 * n * c["vocab"]}
    lengths = _lengths(c)
    tables = 4 * sum((n + c["page"] - 1) // c["page"] for n in lengths)
    if c["kind"] == "bounds":
        tokens = sum(lengths) if c["new"] > 1 else c["batch"]
        pages = sum((n + c["page"] - 1) // c["page"] for n in lengths) if c["new"] > 1 else c["batch"]
        k = tokens * c["kv"] * c["dim"]
        rows = 2 * tokens * c["kv"] * _row(c)
        b = 2 * k * _size(c["dtype"]) + rows + 8 * tokens + tables + (1 if c["new"] > 1 else 2) * pages * c["kv"] * _bounds_row(c)
        if _size(c["cache"]) == 1:
            b += rows + 2 * k * _size(c["dtype"])       # read back
        return {"bytes": b, "flops": 8 * k}
    tokens = c["batch"] * c["new"]
    q = tokens * c["heads"] * c["dim"] * _size(c["dtype"])
    if c["kind"] == "shared":
        pairs, first = 0, c["prefix"]
        for n in lengths:
            for p in range(max(c["prefix"] + n - c["new"], 0), c["prefix"] + n):
                lo = max(p + 1 - c["window"], 0) if c["window"] else 0
                pairs += p + 1 - lo
                first = min(first, lo)
        seen = c["prefix"] - first + sum(min(n, c["window"] + c["new"]) if c["window"] else n for n in lengths)
        return {"bytes": 2 * seen * c["kv"] * _row(c) + 2 * q + 8 * tokens + tables + 4 * (c["prefix"] // c["page"]),
                "flops": 4 * c["heads"] * c["dim"] * pairs}
    blocks = sum((n + c["page"] - 1) // c["page"] for n in lengths)
    pairs = sum(min(n, c["take"] * c["page"]) for n in lengths) * c["new"]
    # each token's own pages are counted, although tokens of a sequence may take the same ones
    return {"bytes": blocks * c["kv"] * _bounds_row(c) + 2 * pairs * c["kv"] * _row(c) + 2 * q + 8 * tokens + tables
            + 4 * tokens * c["kv"] * c["take"],
            "flops": 4 * c["heads"] * c["dim"] * pairs + 4 * c["new"] * blocks * c["kv"] * c["dim"]}


# ------------------------------------------------------------------ inputs
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
        return (x * torch.div(n, m)).round().clamp(-127, 127).to(torch.int8), torch.div(m, n).squeeze(-1)
    frac, e = torch.frexp(amax)
    e = torch.where(frac <= 0.875, e - 9, e - 8).clamp(min=-100)
    return (x * _power(-e)).to(torch.float8_e4m3fn), _power(e).squeeze(-1)


def _pool(c, g, pages):
    """Cache tensors of ``pages`` filled pages: k, v, k_scale, v_scale."""
    shape = (pages, c["kv"], c["page"], c["dim"])
    dt = TYPES[c["cache"]]
    out = [torch.empty(shape, dtype=torch.uint8 if dt.itemsize == 1 else dt, device=DEV).view(dt) for _ in range(2)]
    scales = [torch.empty(shape[:3], device=DEV) if dt.itemsize == 1 else None for _ in range(2)]
    step = max(1, (1 << 26) // (c["kv"] * c["page"] * c["dim"]))
    for i in range(0, pages, step):
        n = min(step, pages - i)
        for t, s, lean in zip(out, scales, (0.5, 0.0)):
            x = torch.randn((n,) + shape[1:], generator=g, device=DEV)
            if lean:
                x += lean * torch.randn((n, c["kv"], 1, c["dim"]), generator=g, device=DEV)
            if s is None:
                t[i:i + step] = x.to(dt)
            else:
                codes, s[i:i + step] = _quantise(x, c["cache"])
                t.view(torch.uint8)[i:i + step] = codes.view(torch.uint8)
    return out + scales


def _held(t, s, idx):
    """f32 values that the cache holds in pages idx."""
    if s is None:
        return t[idx].float()
    return t.view(torch.uint8)[idx].view(t.dtype).float() * s[idx][..., None]


def _all_bounds(c, pool, last):
    """Bounds [pages, kv, 2, dim] of all pages; ``last``: each page's last written row."""
    k, ks = pool[0], pool[2]
    out = torch.empty(k.shape[0], c["kv"], 2, c["dim"], dtype=torch.float32 if ks is not None else k.dtype, device=DEV)
    row = torch.arange(c["page"], device=DEV)[None, None, :, None]
    step = max(1, (1 << 26) // (c["kv"] * c["page"] * c["dim"]))
    for i in range(0, k.shape[0], step):
        idx = torch.arange(i, min(i + step, k.shape[0]), device=DEV)
        x, past = _held(k, ks, idx), row > last[idx][:, None, None, None]
        out[idx, :, 0] = x.masked_fill(past, math.inf).amin(2).to(out.dtype)
        out[idx, :, 1] = x.masked_fill(past, -math.inf).amax(2).to(out.dtype)
    return out


def prepare(c, seed):
    g = _gen(seed)
    st = {"case": c}
    if c["kind"] == "verify":
        return _prepare_verify(c, g, st)
    lengths = _lengths(c)
    front = c["prefix"] // c["page"] if c["kind"] == "shared" else 0
    need = [front + (n + c["page"] - 1) // c["page"] for n in lengths]
    pages = front + sum(n - front for n in need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["batch"], max(need)), -1, dtype=torch.int32, device=DEV)
    table[:, :front] = order[:front]
    last = torch.full((pages,), c["page"] - 1, device=DEV)
    at = front
    for b, n in enumerate(need):
        table[b, front:n] = order[at:at + n - front]
        at += n - front
        last[table[b, n - 1].long()] = (lengths[b] - 1) % c["page"]
    st["table"], st["pool"], st["front"] = table, _pool(c, g, pages), front
    ends = torch.tensor(lengths, device=DEV) + front * c["page"]
    if c["kind"] == "bounds" and c["new"] > 1:
        p = torch.arange(max(lengths), device=DEV).expand(c["batch"], -1)
        st["positions"] = torch.where(p < ends[:, None], p, -1)      # shorter prompts are padded
    else:
        st["positions"] = (ends[:, None] - c["new"] + torch.arange(c["new"], device=DEV)).clamp(min=-1)
    shape = tuple(st["positions"].shape)
    dt = TYPES[c["dtype"]]
    if c["kind"] == "bounds":
        # keys and values as a projection gives them: one row of k|v a token
        kv = _normal(g, shape + (2 * c["kv"], c["dim"]), dt)
        st["k"], st["v"] = kv[..., :c["kv"], :], kv[..., c["kv"]:, :]
        st["bounds"] = torch.zeros(pages, c["kv"], 2, c["dim"], device=DEV,
                                   dtype=st["pool"][0].dtype if st["pool"][2] is None else torch.float32)
        if c["new"] == 1:       # of what the sequences held before
            st["bounds"] = _all_bounds(c, st["pool"], last)
    else:
        st["q"] = _normal(g, shape + (c["heads"], c["dim"]), dt, 2.0)
        if c["kind"] == "select":
            st["bounds"] = _all_bounds(c, st["pool"], last)
    if own:
        _handle(st)
    return st


def _prepare_verify(c, g, st):
    """Probabilities of both models over the vocabulary, tokens drawn from the draft's; some sequences have fewer."""
    B, n, V, dt = c["batch"], c["drafted"], c["vocab"], TYPES[c["dtype"]]
    target = torch.empty(B, n + 1, V, dtype=dt, device=DEV)
    draft = torch.empty(B, n, V, dtype=dt, device=DEV) if c["draft"] else None
    drafted = torch.empty(B, n, dtype=torch.int64, device=DEV)
    for b in range(B):
        logits = torch.randn(n + 1, V, generator=g, device=DEV) * 2.5
        target[b] = torch.softmax(logits, -1).to(dt)
        near = torch.softmax(logits[:n] + 0.5 * torch.randn(n, V, generator=g, device=DEV), -1)
        if draft is not None:
            draft[b] = near.to(dt)
        noise = torch.rand(n, V, generator=g, device=DEV).clamp(min=1e-10)
        drafted[b] = (near.clamp(min=1e-30).log() - (-noise.log()).log()).argmax(-1)     # a token of that probability
    count = torch.randint(max(n - 2, 0), n + 1, (B,), generator=g, device=DEV)
    count[0] = n
    drafted[torch.arange(n, device=DEV) >= count[:, None]] = -1
    st.update(target=target, draft=draft, drafted=drafted,
              uniforms=torch.rand(B, n + 1, generator=g, device=DEV))
    if not c["draft"]:      # tokens that the target would often give
        top = target[:, :n].argmax(-1)
        st["drafted"] = torch.where((drafted >= 0) & (torch.rand(B, n, generator=g, device=DEV) < 0.7), top, drafted)
    return st


def _epure():
    path = os.path.join(_ROOT, "epure-runtime_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import epure
    return epure


def _handle(st):
    if "cache" not in st:
        st["cache"] = _epure().PagedKVCache.of(*st["pool"], k_bounds=st.get("bounds"))
    return st["cache"]


# ------------------------------------------------------------------ plain forms
def _context(t, s, table):
    """All pages of every sequence in order, f32 [batch, kv, positions, dim]."""
    x = _held(t, s, table.long().clamp(min=0))
    b, w, h, p, d = x.shape
    return x.transpose(1, 2).reshape(b, h, w * p, d)


def _part(qh, k, v, ok, scale):
    """Maximum, sum and output of one stretch of positions; qh [.., rows, d], k and v [.., L, d], ok [.., rows, L]."""
    s = torch.matmul(qh, k.transpose(-1, -2)) * scale
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - m.clamp(min=torch.finfo(torch.float32).min))
    return m, e.sum(-1, keepdim=True), torch.matmul(e, v)


def _plain_shared(c, st):
    q, pos, pool, front = st["q"], st["positions"], st["pool"], st["front"]
    b, n, heads, d = q.shape
    kv, g, P, scale = c["kv"], heads // c["kv"], front * c["page"], d ** -0.5
    qh = q.float().view(b, n, kv, g, d).permute(2, 0, 1, 3, 4)          # kv, b, n, g, d

    def seen(j):        # b, n, 1, L
        ok = j <= pos[..., None]
        return (ok & (j > pos[..., None] - c["window"]) if c["window"] else ok)[:, :, None, :]

    # the shared pages, once for all rows of a key head
    k, v = (_context(t, s, st["table"][:1, :front])[0] for t, s in zip(pool[:2], pool[2:]))
    ok = seen(torch.arange(P, device=DEV)).expand(b, n, g, P).reshape(1, b * n * g, P)
    m0, l0, o0 = (x.view(kv, b, n, g, -1) for x in _part(qh.reshape(kv, b * n * g, d), k, v, ok, scale))
    del k, v, ok
    # each sequence's own
    k, v = (_context(t, s, st["table"][:, front:]) for t, s in zip(pool[:2], pool[2:]))
    ok = seen(P + torch.arange(k.shape[2], device=DEV)).expand(b, n, g, -1).reshape(b, 1, n * g, -1)
    own_rows = qh.permute(1, 0, 2, 3, 4).reshape(b, kv, n * g, d)
    m1, l1, o1 = (x.view(b, kv, n, g, -1).transpose(0, 1) for x in _part(own_rows, k, v, ok, scale))
    m = torch.maximum(m0, m1).clamp(min=torch.finfo(torch.float32).min)
    f0, f1 = torch.exp(m0 - m), torch.exp(m1 - m)
    total = l0 * f0 + l1 * f1
    o = (o0 * f0 + o1 * f1) / torch.where(total > 0, total, 1.0)
    return o.permute(1, 2, 0, 3, 4).reshape(b, n, heads, d).to(q.dtype)


def _plain_bounds(c, st):
    pos, pool, bounds = st["positions"], st["pool"], st["bounds"]
    p = pos.clamp(min=0)
    page, row = st["table"].long().gather(1, p // c["page"]).clamp(min=0), p % c["page"]
    at = pos >= 0
    real = (lambda x: x[at]) if c["new"] > 1 else (lambda x: x.flatten(0, 1))   # one token: no padding
    pg, rw = real(page), real(row)
    for x, t, s in ((st["k"], pool[0], pool[2]), (st["v"], pool[1], pool[3])):
        x = real(x).float()
        if s is None:
            t[pg, :, rw] = x.to(t.dtype)
        else:
            codes, scale = _quantise(x, c["cache"])
            t.view(torch.uint8)[pg, :, rw] = codes.view(torch.uint8)
            s[pg, :, rw] = scale
    # pages that were written, with the last row of each
    if c["new"] > 1:
        first = torch.arange(0, pos.shape[1], c["page"], device=DEV)
        ends = pos.amax(1, keepdim=True)
        used = first <= ends
        pages = st["table"].long()[:, :first.shape[0]][used]
        last = (ends - first).clamp(max=c["page"] - 1)[used]
    else:
        pages, last = pg, rw
    x = _held(pool[0], pool[2], pages)
    past = torch.arange(c["page"], device=DEV)[None, None, :, None] > last[:, None, None, None]
    bounds[pages, :, 0] = x.masked_fill(past, math.inf).amin(2).to(bounds.dtype)
    bounds[pages, :, 1] = x.masked_fill(past, -math.inf).amax(2).to(bounds.dtype)
    if pool[2] is None:
        return [pool[0], pool[1], bounds]
    out = []
    for t, s in zip(pool[:2], pool[2:]):
        x = t.view(torch.uint8)[page, :, row].view(t.dtype).float() * s[page, :, row][..., None]
        out.append(torch.where(at[:, :, None, None], x, 0.0).to(TYPES[c["dtype"]]))
    return out + [bounds]


def _plain_select(c, st):
    q, pos, pool, table = st["q"], st["positions"], st["pool"], st["table"].long().clamp(min=0)
    b, n, heads, d = q.shape
    kv, g = c["kv"], heads // c["kv"]
    # scores in 64 bits: pages next to the border are told apart exactly
    qd = q.double().view(b, n, kv, g, d).transpose(1, 2)                 # b, kv, n, g, d
    up, down = qd.clamp(min=0).sum(3), qd.clamp(max=0).sum(3)
    bounds = st["bounds"][table].double()                               # b, w, kv, 2, d
    score = torch.matmul(up, bounds[:, :, :, 1].permute(0, 2, 3, 1).contiguous())
    score += torch.matmul(down, bounds[:, :, :, 0].permute(0, 2, 3, 1).contiguous())
    del bounds
    j = torch.arange(score.shape[-1], device=DEV)
    mine = (pos // c["page"])[:, None, :, None]
    score = torch.where(j == mine, math.inf, torch.where(j < mine, score, -math.inf))
    score, order = torch.sort(score, dim=-1, descending=True, stable=True)
    w = min(c["take"], order.shape[-1])
    order, score = order[..., :w], score[..., :w]
    order = torch.where((score > -math.inf) & (pos[:, None, :, None] >= 0), order, torch.iinfo(torch.int32).max)
    order = torch.nn.functional.pad(order, (0, c["take"] - w), value=torch.iinfo(torch.int32).max).sort(-1).values
    blocks = torch.where(order == torch.iinfo(torch.int32).max, -1, order).transpose(1, 2)     # b, n, kv, take
    # attention over them
    idx = torch.where(blocks >= 0, table.gather(1, blocks.clamp(min=0).flatten(1)).view(blocks.shape), 0)
    h = torch.arange(kv, device=DEV)[None, None, :, None]
    row = blocks.clamp(min=0)[..., None] * c["page"] + torch.arange(c["page"], device=DEV)
    ok = (blocks >= 0)[..., None] & (row <= pos[:, :, None, None, None])
    rows = []
    for t, s in zip(pool[:2], pool[2:]):
        x = t[idx, h].float() if s is None else t.view(torch.uint8)[idx, h].view(t.dtype).float() * s[idx, h][..., None]
        rows.append(x.flatten(3, 4))                                    # b, n, kv, take * page, d
    m, l, o = _part(q.float().view(b, n, kv, g, d), *rows, ok.flatten(3)[:, :, :, None, :], d ** -0.5)
    o = o / torch.where(l > 0, l, 1.0)
    return [blocks.to(torch.int32), o.reshape(b, n, heads, d).to(q.dtype)]


def _plain_verify(c, st):
    target, draft, drafted, u = st["target"], st["draft"], st["drafted"], st["uniforms"].double()
    B, n = drafted.shape
    x = drafted.clamp(min=0)[..., None]
    p = target[:, :n].gather(2, x)[..., 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(2, x)[..., 0].double()
    stands = (drafted >= 0) & (u[:, :n] * q < p)
    accepted = stands.long().cumprod(1).sum(1)
    b = torch.arange(B, device=DEV)
    row = target[b, accepted].double()
    at = accepted.clamp(max=n - 1)
    rejected = (accepted < n) & (drafted[b, at] >= 0)
    if draft is None:
        less = torch.zeros_like(row).scatter_(1, x[b, at], 1.0)
    else:
        less = draft[b, at].double()
    rest = torch.where(rejected[:, None], (row - less).clamp(min=0.0), row)
    rest = torch.where((rest > 0).any(1)[:, None], rest, row)
    run_sum = rest.cumsum(1)
    v = (run_sum <= u[:, n:] * run_sum[:, -1:]).sum(1).clamp(max=c["vocab"] - 1)
    tokens = torch.full((B, n + 1), -1, dtype=torch.int64, device=DEV)
    tokens[:, :n] = torch.where(torch.arange(n, device=DEV) < accepted[:, None], drafted, -1)
    tokens[b, accepted] = v
    return [accepted, tokens]


# ------------------------------------------------------------------ one pass
def run(st):
    c = st["case"]
    if not own:
        return {"shared": _plain_shared, "bounds": _plain_bounds, "select": _plain_select,
                "verify": _plain_verify}[c["kind"]](c, st)
    if c["kind"] == "verify":
        return list(_epure().verify_draft(st["target"], st["drafted"], st["uniforms"], draft=st["draft"]))
    cache, pos, table = _handle(st), st["positions"], st["table"]
    if c["kind"] == "shared":
        return cache.attend(st["q"], pos, table, window=c["window"] or None, shared=st["front"])
    if c["kind"] == "select":
        blocks = cache.select(st["q"], pos, table, c["take"])
        return [blocks, cache.attend(st["q"], pos, table, blocks=blocks)]
    cache.append(st["k"], st["v"], pos, table)
    if st["pool"][2] is None:
        return [cache.k, cache.v, cache.k_bounds]
    return list(cache.read(pos, table, TYPES[c["dtype"]])) + [cache.k_bounds]


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_rows(t, s, pages, h):
    """f64 rows of the given pages of cache head h, in order."""
    if s is None:
        x = t[pages, h].double()
    else:
        x = t.view(torch.uint8)[pages, h].view(t.dtype).double() * s[pages, h].double()[..., None]
    return x.flatten(0, 1)


def _exact_shared(c, st):
    q, pos, pool, front = st["q"].double(), st["positions"].tolist(), st["pool"], st["front"]
    out, g, P = torch.zeros_like(q), c["heads"] // c["kv"], front * c["page"]
    for h in range(c["kv"]):
        common = [_exact_rows(t, s, st["table"][0, :front].long(), h) for t, s in zip(pool[:2], pool[2:])]
        for b, n in enumerate(_lengths(c)):
            pages = st["table"][b, front:front + (n + c["page"] - 1) // c["page"]].long()
            mine = [_exact_rows(t, s, pages, h) for t, s in zip(pool[:2], pool[2:])]
            for i, p in enumerate(pos[b]):
                if p < 0:
                    continue
                lo = max(p + 1 - c["window"], 0) if c["window"] else 0
                k, v = (torch.cat((x[lo:min(P, p + 1)], y[max(lo - P, 0):max(p + 1 - P, 0)])) for x, y in zip(common, mine))
                w = torch.softmax(k @ q[b, i, h * g:(h + 1) * g].T * c["dim"] ** -0.5, 0)
                out[b, i, h * g:(h + 1) * g] = w.T @ v
    return out


def _exact_codes(x, cache):
    """f64 values that 8 bits hold of f64 rows x."""
    m = x.abs().amax(-1, keepdim=True)
    if cache == "int8":
        return (x * 127 / m).round() * (m / 127)
    e = torch.ceil(torch.log2(m / 448))
    e = torch.where(m <= 448 * torch.exp2(e - 1), e - 1, e)
    e = torch.where(m > 448 * torch.exp2(e), e + 1, e)
    y = x * torch.exp2(-e)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)   # spacing of e4m3 at y
    return (y / step).round() * step * torch.exp2(e)


def _exact_bounds(c, st):
    pos, pool, table = st["positions"], st["pool"], st["table"].long()
    eight = pool[2] is not None
    back = [torch.zeros(tuple(pos.shape) + (c["kv"], c["dim"]), dtype=torch.float64, device=DEV) for _ in range(2)]
    whole = [t.double() for t in pool[:2]] if not eight else None
    bounds = st["bounds"].double()
    for b in range(c["batch"]):
        real = pos[b] >= 0
        p = pos[b][real]
        new = [x[b][real].double() for x in (st["k"], st["v"])]
        if eight:
            new = [_exact_codes(x, c["cache"]) for x in new]
        for i in range(2):
            back[i][b][real] = new[i]
            if not eight:
                whole[i][table[b, p // c["page"]], :, p % c["page"]] = new[i]
        for blk in sorted(set((p // c["page"]).tolist())):
            here = p[p // c["page"] == blk]
            r, pg = int(here.max()) % c["page"], int(table[b, blk])
            for h in range(c["kv"]):
                rows = _exact_rows(*(t if t is None else t[pg:pg + 1] for t in (pool[0], pool[2])),
                                   torch.tensor([0], device=DEV), h)
                rows[here % c["page"]] = new[0][p // c["page"] == blk][:, h]
                bounds[pg, h, 0], bounds[pg, h, 1] = rows[:r + 1].amin(0), rows[:r + 1].amax(0)
    return (back if eight else whole) + [bounds]


def _exact_select(c, st):
    q, pos, pool, table = st["q"].double(), st["positions"].tolist(), st["pool"], st["table"].long()
    out, g = torch.zeros_like(q), c["heads"] // c["kv"]
    blocks = torch.full((c["batch"], c["new"], c["kv"], c["take"]), -1, dtype=torch.int32)
    for b in range(c["batch"]):
        for h in range(c["kv"]):
            lim = st["bounds"][table[b].clamp(min=0), h].double()
            for i, p in enumerate(pos[b]):
                if p < 0:
                    continue
                mine = p // c["page"]
                rows = q[b, i, h * g:(h + 1) * g]
                # the larger product of each query value with the page's bounds, one query head after the other
                best = sum(torch.maximum(x * lim[:mine, 0], x * lim[:mine, 1]).sum(1) for x in rows).tolist()
                take = sorted(sorted(range(mine), key=lambda j: (-best[j], j))[:c["take"] - 1] + [mine])
                blocks[b, i, h, :len(take)] = torch.tensor(take, dtype=torch.int32)
                pages = table[b, torch.tensor(take, device=DEV)]
                at = (torch.tensor(take, device=DEV)[:, None] * c["page"] + torch.arange(c["page"], device=DEV)).flatten()
                k, v = (_exact_rows(t, s, pages, h)[at <= p] for t, s in zip(pool[:2], pool[2:]))
                w = torch.softmax(k @ rows.T * c["dim"] ** -0.5, 0)
                out[b, i, h * g:(h + 1) * g] = w.T @ v
    return [blocks.to(DEV), out]


def _exact_verify(c, st):
    drafted, u = st["drafted"].tolist(), st["uniforms"].double().tolist()
    n = c["drafted"]
    accepted, tokens = [], []
    for b in range(c["batch"]):
        k = 0
        while k < n and drafted[b][k] >= 0:
            x = drafted[b][k]
            q = 1.0 if st["draft"] is None else st["draft"][b, k, x].double().item()
            if not u[b][k] * q < st["target"][b, k, x].double().item():
                break
            k += 1
        rest = st["target"][b, k].double().cpu()
        if k < n and drafted[b][k] >= 0:
            less = torch.nn.functional.one_hot(torch.tensor(drafted[b][k]), c["vocab"]).double() \
                if st["draft"] is None else st["draft"][b, k].double().cpu()
            diff = torch.relu(rest - less)
            rest = diff if bool((diff > 0).any()) else rest
        run_sum = torch.cumsum(rest, 0)
        v = int(torch.searchsorted(run_sum, torch.tensor([u[b][n] * run_sum[-1].item()], dtype=torch.float64),
                                   right=True).clamp(max=c["vocab"] - 1))
        accepted.append(k)
        tokens.append(drafted[b][:k] + [v] + [-1] * (n - k))
    return [torch.tensor(accepted, device=DEV), torch.tensor(tokens, device=DEV)]


def exact(c, seed):
    # one key head, sequence and token after the other
    if c["kind"] in ("shared", "select") and c["batch"] * c["new"] * c["kv"] > 4096:
        return None
    st = prepare(c, seed)
    return {"shared": _exact_shared, "bounds": _exact_bounds, "select": _exact_select,
            "verify": _exact_verify}[c["kind"]](c, st)

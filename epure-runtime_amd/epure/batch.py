"""Greedy decode of a ragged batch over the packed linears: the paged
operators of ``epure.paged`` between them.

``epure.decode.Decoder`` runs one sequence in one fused step.  Here any number
of sequences share one pool of pages: a prompt of each is taken in one padded
call (padding has position -1), then every step takes one token a sequence.
Per layer: q, k, v linears, ``PagedKVCache.append`` (the rotation on the way),
``PagedKVCache.attend``, the o linear, and the gated feed-forward pair.  The
residual is float32, what enters and leaves a linear is bfloat16.

What sequences have in common (``share``) is held once and its attention
computed once a step for all of them; with ``select`` a step of few tokens
attends to the pages that matter most to each; drafted tokens are verified
several at a time (``speculate``).

The reference leaves all of this to transformers (epure/runtime.py:373-415).
"""
import torch

from .drafts import verify_draft
from .paged import PagedKVCache, Rotary
from .runtime import PackedLinear


def _rms(x, weight, eps):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()).to(torch.bfloat16)


class BatchDecoder:
    """Decoder over ``epure.decode.DecoderWeights`` for up to ``batch``
    sequences of up to ``max_len`` positions, their keys and values in
    ``n_pages`` pages a layer (default: room for all) of ``cache_dtype``.

    ``select``: calls of up to ``FEW`` new tokens a sequence attend to so many
    pages of each context, chosen anew for every token, layer and cache head
    (``PagedKVCache.select``); longer ones, prompts, to all."""

    FEW = 8

    def __init__(self, weights, batch, max_len, page=64, n_pages=None, cache_dtype=torch.bfloat16, scaling=None,
                 select=None):
        if select is not None and select < 1:
            raise ValueError(f"select takes at least one page, got {select}")
        cfg, dev = weights.cfg, weights.embed.device
        self.w, self.cfg, self.page, self.max_len = weights, cfg, page, max_len
        width = -(-max_len // page)
        self.n_pages = batch * width if n_pages is None else n_pages
        self.rotary = Rotary(cfg.head_dim, max_len, theta=cfg.rope_theta, scaling=scaling, device=dev)
        self.select = None if select is None else min(select, width)     # more pages than a table has: -1 for each
        self.caches = [PagedKVCache(self.n_pages, page, cfg.n_kv, cfg.head_dim, cache_dtype, dev,
                                    bounds=select is not None) for _ in weights.layers]
        self.lin = [{name: PackedLinear(store) for name, store in layer.lin.items()} for layer in weights.layers]
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.reset()

    def reset(self):
        """No sequences, nothing shared; every page is free."""
        self.free = list(range(self.n_pages))
        self.owned = [[] for _ in range(self.table.shape[0])]
        self.shared = 0         # pages that every sequence begins with
        self.lengths = [0] * self.table.shape[0]
        self.table.fill_(-1)

    def release(self, i):
        """Sequence i ends; its own pages are free again."""
        self._trim(i, self.shared * self.page)

    def _more(self, i, n):
        """How many pages n more positions of sequence i take."""
        if self.lengths[i] + n > self.max_len:
            raise ValueError(f"sequence {i}: {self.lengths[i] + n} positions, at most {self.max_len}")
        return -(-(self.lengths[i] + n) // self.page) - self.shared - len(self.owned[i])

    def _grow(self, i, n):
        """Pages for n more positions of sequence i."""
        have, more = self.shared + len(self.owned[i]), self._more(i, n)
        if more > len(self.free):
            raise RuntimeError(f"out of pages: sequence {i} needs {more}, {len(self.free)} are free")
        if more > 0:
            new = [self.free.pop() for _ in range(more)]
            self.owned[i] += new
            self.table[i, have:have + more] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        self.lengths[i] += n

    def _trim(self, i, length):
        """Sequence i goes back to ``length`` positions; pages behind them are free again."""
        keep = max(-(-length // self.page) - self.shared, 0)
        self.free += self.owned[i][keep:]
        del self.owned[i][keep:]
        self.lengths[i] = length
        self.table[i, self.shared + keep:].fill_(-1)

    def _check(self, tokens):
        if any(not 0 <= t < self.cfg.vocab for new in tokens for t in new):
            raise ValueError(f"token ids must lie in [0, {self.cfg.vocab})")

    @torch.no_grad()
    def share(self, tokens):
        """Token ids that all sequences begin with, taken once: their whole
        pages are held once for the batch.  What is left of them (less than a
        page) is returned and begins each sequence's own prompt.  Before any
        sequence has begun."""
        if any(self.lengths):
            raise RuntimeError("a prefix is shared before any sequence has begun")
        n = len(tokens) // self.page
        head, rest = list(tokens[:n * self.page]), list(tokens[n * self.page:])
        self._check([tokens])
        if n * self.page > self.max_len:
            raise ValueError(f"{n * self.page} shared positions, at most {self.max_len}")
        if n > len(self.free):
            raise RuntimeError(f"out of pages: the prefix needs {n}, {len(self.free)} are free")
        if n:
            dev, pages = self.table.device, self.free[-n:]
            row = torch.tensor([pages], dtype=torch.int32, device=dev)
            self._layers(torch.tensor([head], device=dev), torch.arange(n * self.page, device=dev)[None], row, 0)
            del self.free[-n:]
            self.shared, self.lengths = n, [n * self.page] * len(self.lengths)
            self.table[:, :n] = row
        return rest

    def _layers(self, ids, pos, table, shared):
        """float32 [B, S, hidden] behind the last layer; keys and values are stored."""
        cfg, (B, S) = self.cfg, ids.shape
        h = self.w.embed[ids].float()
        for layer, lin, cache in zip(self.w.layers, self.lin, self.caches):
            x = _rms(h, layer.attn_norm, cfg.rms_eps)
            q, k, v = (lin[n](x).view(B, S, -1, cfg.head_dim) for n in ("q", "k", "v"))
            if layer.q_norm is not None:
                q, k = _rms(q, layer.q_norm, cfg.rms_eps), _rms(k, layer.k_norm, cfg.rms_eps)
            q = cache.append(k, v, pos, table, q=q, rotary=self.rotary)
            if self.select is not None and S <= self.FEW:
                o = cache.attend(q, pos, table, blocks=cache.select(q, pos, table, self.select))
            else:
                o = cache.attend(q, pos, table, shared=shared)
            h += lin["o"](o.view(B, S, -1)).float()
            x = _rms(h, layer.mlp_norm, cfg.rms_eps)
            h += lin["down"](torch.nn.functional.silu(lin["gate"](x)) * lin["up"](x)).float()
        return h

    def _logits(self, h):
        return (_rms(h, self.w.final_norm, self.cfg.rms_eps) @ self.w.lm_head.T).float()

    def _take(self, tokens):
        """float32 [B, S, hidden] of new tokens, padded to the longest; their sequences grow."""
        dev = self.table.device
        if len(tokens) > self.table.shape[0]:
            raise ValueError(f"{len(tokens)} sequences in a batch of {self.table.shape[0]}")
        self._check(tokens)
        need = sum(self._more(i, len(t)) for i, t in enumerate(tokens))
        if need > len(self.free):       # before any sequence grows
            raise RuntimeError(f"out of pages: the call needs {need}, {len(self.free)} are free")
        for i, t in enumerate(tokens):
            if len(t) > 0:
                self._grow(i, len(t))
        B, S = len(tokens), max((len(t) for t in tokens), default=0)
        if S == 0:
            return torch.zeros(B, 0, self.w.embed.shape[1], device=dev)
        ids = torch.tensor([list(t) + [0] * (S - len(t)) for t in tokens], device=dev)
        pos = torch.tensor([[*range(self.lengths[i] - len(t), self.lengths[i])] + [-1] * (S - len(t))
                            for i, t in enumerate(tokens)], device=dev)
        return self._layers(ids, pos, self.table[:B], self.shared)

    @torch.no_grad()
    def forward(self, tokens):
        """tokens: one list of new token ids a sequence (empty: none of that
        sequence).  float32 logits [sequences, vocab] after each one's last
        (zeros where it has none)."""
        h, B, dev = self._take(tokens), len(tokens), self.table.device
        if h.shape[1] == 0:
            return torch.zeros(B, self.cfg.vocab, device=dev)
        last = torch.tensor([max(len(t) - 1, 0) for t in tokens], device=dev)
        logits = self._logits(h[torch.arange(B, device=dev), last])
        return logits.masked_fill(torch.tensor([[len(t) == 0] for t in tokens], device=dev), 0.0)

    @torch.no_grad()
    def speculate(self, last, drafts, uniforms=None, draft=None, temperature=1.0):
        """One step over drafted tokens: for each sequence, ``last`` (its
        newest token, not taken yet; None: the sequence is left out) and the
        ids ``drafts[i]`` proposed to follow it.  All are taken in one call,
        verified against the decoder's probabilities at ``temperature``
        (``epure.verify_draft``, which explains ``uniforms`` [B, n + 1] and
        ``draft`` [B, n, vocab], n the longest draft), and those that do not
        stand are taken back.  A list of new tokens a sequence: the drafted
        ones that stand and one more, which is the next call's ``last``."""
        if len(last) != len(drafts):
            raise ValueError(f"{len(last)} sequences, {len(drafts)} drafts")
        if not temperature > 0:
            raise ValueError(f"temperature must be positive, got {temperature}")
        if any(t is None and len(d) > 0 for t, d in zip(last, drafts)):
            raise ValueError("a sequence that is left out has no draft")
        B, n, dev = len(last), max((len(d) for d in drafts), default=0), self.table.device
        if uniforms is None:
            uniforms = torch.rand(B, n + 1, device=dev)
        for name, t, want in (("uniforms", uniforms, (B, n + 1)), ("draft", draft, (B, n, self.cfg.vocab))):
            if t is not None and tuple(t.shape) != want:        # before any sequence grows
                raise ValueError(f"{name} {tuple(t.shape)} must be {list(want)}")
            if t is not None and (t.dtype != torch.float32 or t.device != dev):
                raise TypeError(f"{name} must be float32 on {dev}, got {t.dtype} on {t.device}")
        before = list(self.lengths)
        h = self._take([[] if t is None else [t, *d] for t, d in zip(last, drafts)])
        if h.shape[1] == 0:
            return [[] for _ in last]
        drafted = torch.tensor([[*d] + [-1] * (n - len(d)) for d in drafts], dtype=torch.int64, device=dev).view(B, n)
        target = torch.softmax(self._logits(h) / temperature, -1)
        accepted, tokens = verify_draft(target, drafted, uniforms, draft=draft)
        out = []
        for i, (k, row) in enumerate(zip(accepted.tolist(), tokens.tolist())):
            out.append([] if last[i] is None else row[:k + 1])
            if last[i] is not None:
                self._trim(i, before[i] + 1 + k)
        return out

    def generate(self, prompts, n_new, prefix=()):
        """Greedy continuations of ``prompts`` (lists of token ids, none
        empty), which all follow ``prefix``: a list of n_new ids each."""
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a prompt has at least one token")
        self.reset()
        rest = self.share(prefix)
        out = [[] for _ in prompts]
        new = [rest + list(p) for p in prompts]
        for _ in range(n_new):
            picks = self.forward(new).argmax(-1).tolist()
            for o, t in zip(out, picks):
                o.append(t)
            new = [[t] for t in picks]
        return out

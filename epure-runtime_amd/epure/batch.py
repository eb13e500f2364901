"""Greedy decode of a ragged batch over the packed linears: the paged
operators of ``epure.paged`` between them.

``epure.decode.Decoder`` runs one sequence in one fused step.  Here any number
of sequences share one pool of pages: a prompt of each is taken in one padded
call (padding has position -1), then every step takes one token a sequence.
Per layer: q, k, v linears, ``PagedKVCache.append`` (the rotation on the way),
``PagedKVCache.attend``, the o linear, and the gated feed-forward pair.  The
residual is float32, what enters and leaves a linear is bfloat16.

The reference leaves all of this to transformers (epure/runtime.py:373-415).
"""
import torch

from .paged import PagedKVCache, Rotary
from .runtime import PackedLinear


def _rms(x, weight, eps):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()).to(torch.bfloat16)


class BatchDecoder:
    """Decoder over ``epure.decode.DecoderWeights`` for up to ``batch``
    sequences of up to ``max_len`` positions, their keys and values in
    ``n_pages`` pages a layer (default: room for all) of ``cache_dtype``."""

    def __init__(self, weights, batch, max_len, page=64, n_pages=None, cache_dtype=torch.bfloat16, scaling=None):
        cfg, dev = weights.cfg, weights.embed.device
        self.w, self.cfg, self.page, self.max_len = weights, cfg, page, max_len
        width = -(-max_len // page)
        self.n_pages = batch * width if n_pages is None else n_pages
        self.rotary = Rotary(cfg.head_dim, max_len, theta=cfg.rope_theta, scaling=scaling, device=dev)
        self.caches = [PagedKVCache(self.n_pages, page, cfg.n_kv, cfg.head_dim, cache_dtype, dev)
                       for _ in weights.layers]
        self.lin = [{name: PackedLinear(store) for name, store in layer.lin.items()} for layer in weights.layers]
        self.table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
        self.reset()

    def reset(self):
        """No sequences; every page is free."""
        self.free = list(range(self.n_pages))
        self.owned = [[] for _ in range(self.table.shape[0])]
        self.lengths = [0] * self.table.shape[0]
        self.table.fill_(-1)

    def release(self, i):
        """Sequence i ends; its pages are free again."""
        self.free += self.owned[i]
        self.owned[i], self.lengths[i] = [], 0
        self.table[i].fill_(-1)

    def _more(self, i, n):
        """How many pages n more positions of sequence i take."""
        if self.lengths[i] + n > self.max_len:
            raise ValueError(f"sequence {i}: {self.lengths[i] + n} positions, at most {self.max_len}")
        return -(-(self.lengths[i] + n) // self.page) - len(self.owned[i])

    def _grow(self, i, n):
        """Pages for n more positions of sequence i."""
        have, more = len(self.owned[i]), self._more(i, n)
        if more > len(self.free):
            raise RuntimeError(f"out of pages: sequence {i} needs {more}, {len(self.free)} are free")
        if more > 0:
            new = [self.free.pop() for _ in range(more)]
            self.owned[i] += new
            self.table[i, have:have + more] = torch.tensor(new, dtype=torch.int32, device=self.table.device)
        self.lengths[i] += n

    @torch.no_grad()
    def forward(self, tokens):
        """tokens: one list of new token ids a sequence (empty: none of that
        sequence).  float32 logits [sequences, vocab] after each one's last
        (zeros where it has none)."""
        dev, cfg = self.table.device, self.cfg
        if len(tokens) > self.table.shape[0]:
            raise ValueError(f"{len(tokens)} sequences in a batch of {self.table.shape[0]}")
        if any(not 0 <= t < cfg.vocab for new in tokens for t in new):
            raise ValueError(f"token ids must lie in [0, {cfg.vocab})")
        need = sum(self._more(i, len(t)) for i, t in enumerate(tokens))
        if need > len(self.free):       # before any sequence grows
            raise RuntimeError(f"out of pages: the call needs {need}, {len(self.free)} are free")
        for i, t in enumerate(tokens):
            if len(t) > 0:
                self._grow(i, len(t))
        B, S = len(tokens), max((len(t) for t in tokens), default=0)
        if S == 0:
            return torch.zeros(B, cfg.vocab, device=dev)
        ids = torch.tensor([list(t) + [0] * (S - len(t)) for t in tokens], device=dev)
        pos = torch.tensor([[*range(self.lengths[i] - len(t), self.lengths[i])] + [-1] * (S - len(t))
                            for i, t in enumerate(tokens)], device=dev)
        table = self.table[:B]
        h = self.w.embed[ids].float()
        for layer, lin, cache in zip(self.w.layers, self.lin, self.caches):
            x = _rms(h, layer.attn_norm, cfg.rms_eps)
            q, k, v = (lin[n](x).view(B, S, -1, cfg.head_dim) for n in ("q", "k", "v"))
            if layer.q_norm is not None:
                q, k = _rms(q, layer.q_norm, cfg.rms_eps), _rms(k, layer.k_norm, cfg.rms_eps)
            q = cache.append(k, v, pos, table, q=q, rotary=self.rotary)
            h += lin["o"](cache.attend(q, pos, table).view(B, S, -1)).float()
            x = _rms(h, layer.mlp_norm, cfg.rms_eps)
            h += lin["down"](torch.nn.functional.silu(lin["gate"](x)) * lin["up"](x)).float()
        last = torch.tensor([max(len(t) - 1, 0) for t in tokens], device=dev)
        x = _rms(h[torch.arange(B, device=dev), last], self.w.final_norm, cfg.rms_eps)
        logits = (x @ self.w.lm_head.T).float()
        return logits.masked_fill(torch.tensor([[len(t) == 0] for t in tokens], device=dev), 0.0)

    def generate(self, prompts, n_new):
        """Greedy continuations of ``prompts`` (lists of token ids, none
        empty): a list of n_new ids each."""
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a prompt has at least one token")
        self.reset()
        out = [[] for _ in prompts]
        new = [list(p) for p in prompts]
        for _ in range(n_new):
            picks = self.forward(new).argmax(-1).tolist()
            for o, t in zip(out, picks):
                o.append(t)
            new = [[t] for t in picks]
        return out

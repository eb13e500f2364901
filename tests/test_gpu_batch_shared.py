"""BatchDecoder with a shared prefix, selected pages and drafted tokens: the
three together over the packed linears, against the float32 decoder of
oracle/decoder.py one sequence at a time."""
import pytest
import torch

from epure.batch import BatchDecoder
from epure.decode import DecoderConfig, random_weights
from oracle import drafts as od
from oracle.decoder import RefDecoder

DEV = torch.device("cuda:0")
CFG = DecoderConfig(512, 1024, 2, 8, 2, 64, 1000, 5e5)
HELD = {torch.bfloat16: 0.0, torch.int8: 2.7 / 254, torch.float8_e4m3fn: 2.0 ** -4}


def tolerance(cache_dtype):
    """As for a ragged batch without sharing: a layer rounds to bf16 some ten
    times on the way of a value, a cache row of 8 bits is off by HELD of one."""
    return CFG.layers * (10 * 2.0 ** -8 + 2 * HELD[cache_dtype]) + 2 * 2.0 ** -8


def ids(g, n):
    return torch.randint(0, CFG.vocab, (n,), generator=g).tolist()


class Refs:
    """One RefDecoder a sequence."""

    def __init__(self, w, n):
        self.refs, self.at = [RefDecoder.from_weights(w, 200) for _ in range(n)], [0] * n

    def take(self, i, tokens):
        for t in tokens:
            out = self.refs[i].step(t, self.at[i])
            self.at[i] += 1
        return out

    def back(self, i, n):
        self.at[i] -= n         # positions behind are written again before they are read


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", list(HELD))
@pytest.mark.parametrize("select", [None, 12])
def test_logits_behind_a_shared_prefix(cache_dtype, select):
    """With ``select`` no fewer pages than there are: the same attention through the list."""
    w = random_weights(CFG, seed=3, device=DEV)
    d = BatchDecoder(w, 3, 192, page=16, cache_dtype=cache_dtype, select=select)
    g = torch.Generator().manual_seed(1)
    prefix, prompts = ids(g, 75), [ids(g, n) for n in (20, 1, 9)]
    rest = d.share(prefix)
    assert rest == prefix[64:] and d.shared == 4 and d.lengths == [64] * 3
    assert (d.table[:, :4] == d.table[:1, :4]).all() and len(d.free) == d.n_pages - 4
    refs = Refs(w, 3)
    for i in range(3):
        refs.take(i, prefix[:64])
    steps = [[rest + p for p in prompts]] + [[ids(g, 1) for _ in range(3)] for _ in range(4)]
    steps[2][1] = []
    for new in steps:
        got = d.forward(new)
        for i, t in enumerate(new):
            if not t:
                assert (got[i] == 0).all()
                continue
            want = refs.take(i, t)
            assert (got[i] - want).norm() <= tolerance(cache_dtype) * want.norm()
    d.release(1)
    assert d.lengths[1] == 64 and d.owned[1] == [] and (d.table[1, 4:] == -1).all() and (d.table[1, :4] >= 0).all()
    got = d.forward([[], prompts[2]])
    refs.back(1, refs.at[1] - 64)
    want = refs.take(1, prompts[2])
    assert (got[1] - want).norm() <= tolerance(cache_dtype) * want.norm()


@pytest.mark.gpu
def test_a_generation_behind_a_prefix_takes_its_pages_once():
    """Greedy picks of close logits may differ where sums are taken in another order: the first is compared by its logits."""
    w = random_weights(CFG, seed=5, device=DEV)
    g = torch.Generator().manual_seed(3)
    prefix, prompts = ids(g, 70), [ids(g, 5), ids(g, 30), ids(g, 1)]
    d = BatchDecoder(w, 3, 128, page=16, n_pages=4 + 3 * 3)      # without sharing: 5 + 7 + 5
    out = d.generate(prompts, 6, prefix=prefix)
    assert [len(o) for o in out] == [6, 6, 6] and d.shared == 4
    assert d.generate(prompts, 6, prefix=prefix) == out
    refs = Refs(w, 3)
    for i in range(3):
        want = refs.take(i, prefix + prompts[i])
        assert want[out[i][0]] >= want.max() - 2 * tolerance(torch.bfloat16) * want.norm()


@pytest.mark.gpu
@pytest.mark.parametrize("cache_dtype", list(HELD))
def test_a_long_prefix_gives_what_it_gives_each_sequence(cache_dtype):
    """1040 positions in common (computed once a step) against the same tokens in
    every sequence: twice a decoder's distance from float32."""
    w = random_weights(CFG, seed=6, device=DEV)
    g = torch.Generator().manual_seed(4)
    prefix, prompts = ids(g, 1045), [ids(g, n) for n in (12, 1, 30, 4)]
    shared, apart = (BatchDecoder(w, 4, 1200, page=16, cache_dtype=cache_dtype) for _ in range(2))
    rest = shared.share(prefix)
    assert len(rest) == 5 and shared.shared == 65
    new, whole = [rest + p for p in prompts], [prefix + p for p in prompts]
    for _ in range(4):
        got, want = shared.forward(new), apart.forward(whole)
        assert ((got - want).norm(dim=-1) <= 2 * tolerance(cache_dtype) * want.norm(dim=-1)).all()
        new = whole = [ids(g, 1) for _ in range(4)]
    assert shared.lengths == apart.lengths and len(shared.free) == shared.n_pages - 65 - sum(map(len, shared.owned))


@pytest.mark.gpu
@pytest.mark.parametrize("select", [None, 3])
def test_drafted_tokens_stand_or_are_taken_back(select):
    """Against the oracle on the same probabilities (a twin's, taken token by
    token), lengths and pages behind them, and the logits of a later step."""
    w = random_weights(CFG, seed=4, device=DEV)
    d = BatchDecoder(w, 3, 160, page=16, select=select)
    g = torch.Generator().manual_seed(2)
    rest = d.share(ids(g, 32))
    prompts = [rest + ids(g, n) for n in (14, 3, 31)]
    last = d.forward(prompts).argmax(-1).tolist()
    for step in range(4):
        lengths = list(d.lengths)
        first = [1 - (step == 2), 1, 1]
        # what the decoder gives token by token, and back
        drafts = [[], [], []]
        for i in range(3):
            if first[i]:
                t = last[i]
                for _ in range(1 + (i + step) % 3):
                    new = [[], [], []]
                    new[i] = [t]
                    t = d.forward(new)[i].argmax().item()
                    drafts[i].append(t)
                d._trim(i, lengths[i])
        if step == 1:
            drafts[0][-1] = (drafts[0][-1] + 1) % CFG.vocab      # one that will not stand
        n = max(map(len, drafts))
        u = torch.full((3, n + 1), 0.5, device=DEV)
        out = d.speculate([t if f else None for t, f in zip(last, first)], drafts, u, temperature=1e-3)
        for i in range(3):
            if not first[i]:
                assert out[i] == [] and d.lengths[i] == lengths[i]
                continue
            k = len(out[i]) - 1
            assert out[i][:k] == drafts[i][:k] and k <= len(drafts[i])
            assert d.lengths[i] == lengths[i] + 1 + k
            assert len(d.owned[i]) == -(-d.lengths[i] // 16) - 2 and (d.table[i, 2 + len(d.owned[i]):] == -1).all()
            last[i] = out[i][-1]
        if step == 1:
            assert len(out[0]) <= len(drafts[0])
    assert len(d.free) + sum(map(len, d.owned)) + 2 == d.n_pages and len(set(d.free) | set(sum(d.owned, []))) == d.n_pages - 2


@pytest.mark.gpu
def test_a_step_verifies_as_the_oracle_does():
    w = random_weights(CFG, seed=4, device=DEV)
    g = torch.Generator().manual_seed(5)
    prompts, last, drafts = [ids(g, 7), ids(g, 40)], [11, 12], [ids(g, 3), ids(g, 2)]
    twin = BatchDecoder(w, 2, 96, page=16)
    twin.forward(prompts)
    h = twin._take([[t] + x for t, x in zip(last, drafts)])
    target = torch.softmax(twin._logits(h) / 0.7, -1)
    draft = torch.full((2, 3, CFG.vocab), 1.0 / CFG.vocab, device=DEV)
    drafted = torch.tensor([drafts[0], drafts[1] + [-1]])
    for seed in range(6):
        u = torch.rand(2, 4, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV)
        d = BatchDecoder(w, 2, 96, page=16)
        d.forward(prompts)
        got = d.speculate(last, drafts, u, draft=draft, temperature=0.7)
        k, tokens = od.verify(target, drafted, u, draft)
        assert got == [t[:n + 1] for t, n in zip(tokens, k)]


# ------------------------------------------------------------------ on the host
def small(**more):
    w = random_weights(DecoderConfig(256, 256, 1, 2, 1, 64, 50, 1e4), device="cpu")
    return BatchDecoder(w, 2, 64, page=16, n_pages=6, **more)


def test_pages_of_sequences_behind_a_prefix():
    d = small()
    d.shared, d.lengths, d.free = 2, [32, 32], [0, 1, 2, 3]
    d.table[:, :2] = torch.tensor([5, 4])
    d._grow(0, 1)
    assert d.owned[0] == [3] and d.table[0].tolist() == [5, 4, 3, -1]
    d._grow(0, 31)
    assert d.lengths[0] == 64 and len(d.owned[0]) == 2
    d._trim(0, 48)
    assert d.owned[0] == [3] and d.table[0].tolist() == [5, 4, 3, -1] and d.free == [0, 1, 2]
    d._trim(0, 33)
    assert d.owned[0] == [3]
    d.release(0)
    assert d.lengths == [32, 32] and sorted(d.free) == [0, 1, 2, 3] and d.table[0].tolist() == [5, 4, -1, -1]
    d.reset()
    assert d.shared == 0 and len(d.free) == 6 and (d.table == -1).all()


def test_refusals_change_nothing():
    d = small()
    assert d.share([1] * 15) == [1] * 15 and d.shared == 0
    for bad, error in (([1] * 80, ValueError), ([50] * 16, ValueError), ([-1], ValueError)):
        with pytest.raises(error):
            d.share(bad)
    d.free = [0]
    with pytest.raises(RuntimeError, match="out of pages"):
        d.share([1] * 32)
    d.reset()
    d._grow(1, 3)
    with pytest.raises(RuntimeError, match="before any"):
        d.share([1] * 16)
    for args, error in ((([1], [[], []]), ValueError), (([1, None], [[], [2]]), ValueError),
                        (([1, 2], [[], []], None, None, 0.0), ValueError),
                        (([1, 2], [[3], []], torch.zeros(2, 3)), ValueError),
                        (([1, 2], [[3], []], None, torch.zeros(2, 1, 49)), ValueError),
                        (([1, 2], [[3], []], torch.zeros(2, 2).double()), TypeError),
                        (([1, 2], [[3], []], None, torch.zeros(2, 1, 50).half()), TypeError),
                        (([1, 50], [[], []]), ValueError), (([1] * 3, [[]] * 3), ValueError),
                        (([1, 2], [[3] * 64, []]), ValueError)):
        with pytest.raises(error):
            d.speculate(*args)
        assert d.lengths == [0, 3] and len(d.free) == 5
    assert d.speculate([None, None], [[], []]) == [[], []]
    with pytest.raises(ValueError):
        small(select=0)

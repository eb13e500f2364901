"""A ragged batch through BatchDecoder: packed linears, rotations, the paged
cache and attention over it together, against the float32 decoder of
oracle/decoder.py one sequence at a time."""
import pytest
import torch

from epure.batch import BatchDecoder
from epure.decode import DecoderConfig, random_weights
from oracle.decoder import RefDecoder

CFGS = [DecoderConfig(512, 1024, 2, 8, 2, 64, 1000, 5e5),
        DecoderConfig(512, 1024, 2, 4, 4, 128, 1000, 1e6, 1e-6, qk_norm=True, tie_embeddings=True)]


def test_batch_refuses_and_hands_pages_back():
    w = random_weights(DecoderConfig(256, 256, 1, 2, 1, 64, 50, 1e4), device="cpu")
    d = BatchDecoder(w, 2, 64, page=16, n_pages=5)
    d._grow(0, 33)
    assert len(d.owned[0]) == 3 and d.table[0].tolist()[:3] == d.owned[0] and d.table[0, 3] == -1
    d._grow(0, 15)
    assert len(d.owned[0]) == 3 and d.lengths[0] == 48
    with pytest.raises(RuntimeError, match="out of pages"):
        d._grow(1, 33)
    with pytest.raises(ValueError, match="at most"):
        d._grow(0, 17)
    assert d.lengths == [48, 0]
    d.release(0)
    assert sorted(d.free) == list(range(5)) and (d.table == -1).all()
    with pytest.raises(ValueError):
        d.generate([[1], []], 2)
    with pytest.raises(ValueError):
        d.forward([[1]] * 3)


@pytest.mark.gpu
@pytest.mark.parametrize("cfg", CFGS)
@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.int8, torch.float8_e4m3fn])
def test_logits_of_a_ragged_batch(cfg, cache_dtype):
    """Norm-wise: a layer rounds to bf16 some ten times on the way of a value
    (half a step each, 2^-8), a cache row of 8 bits is off by up to
    2.7 / 254 (int8: half a step at a row's usual largest of 2.7 standard
    deviations) or 2^-4 (e4m3) of a value, keys and values each; two layers
    and the head's input, added up."""
    dev = torch.device("cuda:0")
    w = random_weights(cfg, seed=3, device=dev)
    held = {torch.bfloat16: 0.0, torch.int8: 2.7 / 254, torch.float8_e4m3fn: 2.0 ** -4}[cache_dtype]
    tol = cfg.layers * (10 * 2.0 ** -8 + 2 * held) + 2 * 2.0 ** -8
    d = BatchDecoder(w, 3, 96, page=16, cache_dtype=cache_dtype)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g).tolist() for n in (37, 1, 16)]
    steps = [prompts] + [[[t] for t in torch.randint(0, cfg.vocab, (3,), generator=g).tolist()] for _ in range(6)]
    steps[3] = [steps[3][0], [], steps[3][2]]          # a step without one of the sequences
    refs, at = [RefDecoder.from_weights(w, 96) for _ in range(3)], [0, 0, 0]
    for new in steps:
        got = d.forward(new)
        for i, toks in enumerate(new):
            if not toks:
                assert (got[i] == 0).all()
                continue
            for t in toks:
                want = refs[i].step(t, at[i])
                at[i] += 1
            err = (got[i] - want).norm() / want.norm()
            assert err <= tol, f"sequence {i}, position {at[i] - 1}: {err.item():.4f} > {tol:.4f}"
    assert d.lengths == at


@pytest.mark.gpu
def test_a_sequence_does_not_depend_on_the_pages_it_gets():
    dev = torch.device("cuda:0")
    w = random_weights(CFGS[0], seed=4, device=dev)
    d = BatchDecoder(w, 2, 128, page=16, n_pages=12)
    prompts = [[5, 6, 7] * 9, [1, 2]]
    first = d.generate(prompts, 8)
    d.forward([[9] * 40, []])
    d.release(0)
    keep = d.free
    again = d.generate(prompts, 8)
    d.reset()
    d.free = keep[::-1]
    assert again == first
    assert all(len(o) == 8 for o in first)


def test_a_call_that_does_not_fit_changes_nothing():
    w = random_weights(DecoderConfig(256, 256, 1, 2, 1, 64, 50, 1e4), device="cpu")
    d = BatchDecoder(w, 3, 64, page=16, n_pages=5)
    d._grow(1, 16)
    table = d.table.clone()
    for bad, error in (([[1] * 33, [], [1] * 33], RuntimeError),     # 6 pages of 4
                       ([[1], [1] * 49], ValueError),                # past max_len
                       ([[1], [50]], ValueError), ([[1], [3, -1]], ValueError)):
        with pytest.raises(error):
            d.forward(bad)
        assert d.lengths == [0, 16, 0] and len(d.free) == 4 and (d.table == table).all()

"""A batch decoder's sequences on pages in another order."""
import pytest
import torch

from epure.batch import BatchDecoder
from epure.decode import DecoderConfig, random_weights

pytestmark = pytest.mark.gpu
CFG = DecoderConfig(512, 1024, 2, 8, 2, 64, 1000, 5e5)


@pytest.mark.parametrize("cache_dtype", [torch.bfloat16, torch.int8])
def test_logits_do_not_depend_on_which_pages_a_sequence_gets(cache_dtype):
    """The same calls with the free pages in three orders: the tables differ,
    the logits are equal bit for bit (a sequence's work is cut by its lengths,
    not by its pages)."""
    w = random_weights(CFG, seed=4, device=torch.device("cuda:0"))
    d = BatchDecoder(w, 2, 128, page=16, n_pages=12, cache_dtype=cache_dtype)
    g = torch.Generator().manual_seed(2)
    orders = [list(range(12)), list(range(12))[::-1], torch.randperm(12, generator=g).tolist()]
    steps = [[[5, 6, 7] * 9, [1, 2]], [[9], [8]], [[4] * 30, []], [[3], [2] * 17], [[11], [12]]]
    runs, tables = [], []
    for order in orders:
        d.reset()
        d.free = list(order)
        runs.append([d.forward(new) for new in steps])
        tables.append(d.table.clone())
    for run, table in zip(runs[1:], tables[1:]):
        assert not torch.equal(table, tables[0]) and torch.equal(table < 0, tables[0] < 0)
        for a, b in zip(run, runs[0]):
            assert torch.equal(a, b)

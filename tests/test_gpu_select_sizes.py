"""More pages asked for than there are: none is planned for, and none allocated
before the call is refused."""
import pytest
import torch

from epure import PagedKVCache
from epure.batch import BatchDecoder
from epure.decode import DecoderConfig, random_weights
from epure.kernels import _abi, cuda
from test_gpu_select import BF16, DEV, filled, gen, normal

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _library():
    assert cuda.available()


def test_a_decoder_takes_no_more_pages_than_its_tables_have(monkeypatch):
    w = random_weights(DecoderConfig(512, 1024, 2, 8, 2, 64, 1000, 5e5), seed=3, device=DEV)
    tokens = [[5, 6, 7], [8]]
    want = BatchDecoder(w, 2, 60, page=16, select=4).forward(tokens)
    seen, select = [], PagedKVCache.select

    def record(self, q, positions, table, n):
        seen.append(n)
        return select(self, q, positions, table, n)
    monkeypatch.setattr(PagedKVCache, "select", record)
    got = BatchDecoder(w, 2, 60, page=16, select=1000).forward(tokens)
    assert seen == [4, 4] and torch.equal(got, want)


@pytest.mark.parametrize("native", [True, False])
def test_a_refused_selection_allocates_nothing(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_abi, "call", None)
    g = gen(1)
    cache, table, *_ = filled(g, 2, 3, 16, 1, 64, BF16)
    q, pos = normal(g, 2, 1, 2, 64), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    cache.select(q, pos, table, 2)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for n in (1 << 27, 1 << 40, (0x3fffffff // 16) + 1):
        with pytest.raises(ValueError, match="2\\^30"):
            cache.select(q, pos, table, n)
    assert torch.cuda.max_memory_allocated() - before < 1 << 20

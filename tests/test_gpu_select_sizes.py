"""More pages asked for than there are: none of them is planned for."""
import pytest
import torch

from epure import PagedKVCache
from epure.batch import BatchDecoder
from epure.decode import DecoderConfig, random_weights
from epure.kernels import cuda
from test_gpu_select import DEV

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

"""What an append that keeps bounds refuses before anything is launched."""
import pytest

from epure.kernels import _abi
from test_drafts_cpu import P, cache, heads, tokens

ERR, DTYPE, SHAPE = -1, 1, 2


@pytest.fixture(scope="module")
def lib():
    assert _abi._load() is not None, _abi.LOAD_ERROR
    return _abi.lib


def test_an_append_with_bounds_refuses(lib):
    k, t, c = heads(2, 64), tokens(), cache()
    q32 = _abi.Heads(P, _abi.F32, 4, 256, 256, 64)
    rot = _abi.Rotation(P, P, 10, 64, 0)
    for args, rc in (((None, k, k, None, t, c, None, None), ERR), ((None, k, k, None, t, c, None, P + 8), ERR),
                     ((q32, k, k, None, t, c, P, P), ERR), ((heads(4, 64), k, k, None, t, c, None, P), ERR),
                     ((None, heads(4, 64), k, None, t, c, None, P), ERR), ((None, None, k, None, t, c, None, P), ERR),
                     ((None, k, k, _abi.Rotation(P, P, 10, 66, 0), t, c, None, P), ERR),
                     ((None, k, k, _abi.Rotation(None, P, 10, 64, 0), t, c, None, P), ERR),
                     ((None, k, k, rot, t, cache(page=48), None, P), SHAPE), ((None, k, k, rot, t, cache(dtype=9), None, P), DTYPE),
                     ((None, k, k, rot, tokens(B=1 << 31, S=2), c, None, P), SHAPE)):
        assert lib.ep_kv_append_bounds(*args, None) == rc, args
        assert _abi.last_error()
    assert lib.ep_kv_append_bounds(None, k, k, rot, tokens(B=0), c, None, P, None) == 0
    assert lib.ep_kv_append_bounds(None, k, k, rot, tokens(S=0), c, None, P, None) == 0

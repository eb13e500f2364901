"""Sizes past what the paged operators' launches hold are declined on the
host, before anything is launched (so dummy pointers are never read)."""
import pytest

from epure.kernels import _abi

P, SHAPE = 64, 2


@pytest.fixture(scope="module")
def lib():
    assert _abi._load() is not None, _abi.LOAD_ERROR
    return _abi.lib


def heads(n, d):
    return _abi.Heads(P, _abi.BF16, n, n * d, n * d, d)


def tokens(B, S=1):
    return _abi.Tokens(B, S, P, S, 1, P, 4, 4)


def cache(heads, D, dtype=_abi.BF16):
    return _abi.KVCache(P, P, None, None, dtype, heads, 16, D, 4)


@pytest.mark.parametrize("D,lanes", [(16, 1), (17, 2), (80, 8), (128, 8), (144, 16), (256, 16), (4096, 256)])
def test_rotations_of_too_many_lanes(lib, D, lanes):
    rot = _abi.Rotation(P, P, 16, 16, 0)
    most = (1 << 32) // lanes                           # rows of one launch: fewer
    for q, k, tok in ((1 << 10, 0, tokens(1 << 12, most >> 22)), (4, 0, tokens(most // 4)),
                      (1 << 9, 1 << 9, tokens(most >> 10))):
        rc = lib.ep_rotate(heads(q, D), heads(k, D) if k else None, rot, tok, D, 0, P, P, None)
        assert rc == SHAPE and "more than one launch" in _abi.last_error()


@pytest.mark.parametrize("D,lanes", [(16, 1), (32, 2), (80, 8), (128, 8), (256, 16)])
def test_cache_rows_of_too_many_lanes(lib, D, lanes):
    most = (1 << 32) // lanes
    c = cache(16, D)
    assert lib.ep_kv_read(tokens(most >> 5), c, P, P, _abi.BF16, None) == SHAPE
    assert "more than one launch" in _abi.last_error()
    assert lib.ep_kv_append(None, heads(16, D), heads(16, D), None, tokens(most >> 5), c, None, None) == SHAPE
    assert lib.ep_kv_append(heads(32, D), heads(16, D), heads(16, D), None, tokens(most >> 6), c, P, None) == SHAPE


@pytest.mark.parametrize("q,kv,B,S", [(32, 8, 1 << 20, 64), (32, 1, 1, 1 << 26), (8, 8, 1 << 28, 1), (2, 1, 1, 1 << 29)])
def test_attention_of_too_many_rows(lib, q, kv, B, S):
    rc = lib.ep_paged_attention(heads(q, 64), tokens(B, S), cache(kv, 64), 1.0, 0, P, P, 1 << 62, None)
    assert rc == SHAPE and "more than one call" in _abi.last_error()

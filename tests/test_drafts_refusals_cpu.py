"""The verification of drafted tokens refuses with the code that the header
names for the reason: what is wrong (negative), or what is not served (positive)."""
import ctypes

import pytest

from epure.kernels import _abi
from test_drafts_cpu import P, draft

ARG, WORKSPACE, DTYPE, SHAPE = -1, -3, 1, 2      # EP_ERR_ARG, EP_ERR_WORKSPACE, EP_DECLINE_DTYPE, EP_DECLINE_SHAPE


@pytest.fixture(scope="module")
def lib():
    assert _abi._load() is not None, _abi.LOAD_ERROR
    return _abi.lib


@pytest.mark.parametrize("bad,rc", [
    ({"B": -1}, ARG), ({"V": 0}, ARG), ({"V": -5}, ARG), ({"n": -1}, ARG), ({"target": None}, ARG), ({"drafted": None}, ARG),
    ({"uniforms": None}, ARG), ({"dtype": 7}, DTYPE), ({"dtype": _abi.E4M3}, DTYPE), ({"V": 1 << 40}, SHAPE), ({"V": 1 << 31}, SHAPE),
    ({"n": 1 << 30}, SHAPE), ({"B": 1 << 31}, SHAPE), ({"B": 1 << 30, "V": 1 << 30}, SHAPE)])
def test_the_code_says_why(lib, bad, rc):
    assert lib.ep_verify_draft(ctypes.byref(draft(**bad)), P, P, P, 1 << 62, None) == rc
    assert _abi.last_error()


def test_outputs_and_workspace(lib):
    d = draft()
    n = lib.ep_verify_draft_workspace(ctypes.byref(d))
    for out, tokens, ws, size, rc in ((None, P, P, n, ARG), (P, None, P, n, ARG), (P, P, P + 8, n, SHAPE), (P, P, P, n - 1, WORKSPACE),
                                      (P, P, None, 0, WORKSPACE)):
        assert lib.ep_verify_draft(ctypes.byref(d), out, tokens, ws, size, None) == rc
    assert lib.ep_verify_draft(None, P, P, P, n, None) == ARG

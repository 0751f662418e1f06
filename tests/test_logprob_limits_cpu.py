"""Limits of log probabilities: what a call that is too large, or asks for a number of alternatives below zero, is told before anything touches a
device."""
import ctypes

import numpy as np
import pytest

import mignon_ai_amd as M
from mignon_ai_amd import _lib


def call(n=1, V=8, m=1, k=0):
    buf = (ctypes.c_uint8 * 4096)()  # never read by a refused call
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    rc = _lib.lib().mg_token_logprobs(p, 0, n, V, V, p, m, k, p, p, p, p, None, 0, _lib.MG_PTR_DEVICE, None)
    return rc, _lib.lib().mg_last_error().decode()


@pytest.mark.parametrize("m", [2 ** 30 + 1, 2 ** 31 - 256, 2 ** 31 - 1])
def test_targets_past_what_a_lane_counts_to(m):
    """A lane's targets are 256 apart: its count stays below 2^31."""
    rc, error = call(m=m)
    assert rc == _lib.MG_ERR_INVALID and "shape" in error


def test_rows_past_a_launch():
    """2^24 workgroups: of four short rows, or of one."""
    for n, V in ((2 ** 26, 8), (2 ** 24, 10000)):
        rc, error = call(n=n, V=V)
        assert rc == _lib.MG_ERR_INVALID and "too many rows" in error


@pytest.mark.parametrize("k", [-1, -3, 65, 2 ** 32, 2 ** 32 + 1, -2 ** 32 + 1])
def test_numbers_of_alternatives(k):
    with pytest.raises(M.MignonError, match="k is"):
        M.token_logprobs(np.zeros((2, 100), np.float32), k=k)


@pytest.mark.parametrize("shape", [(2 ** 32 + 3, 1), (2 ** 31, 1), (1, 2 ** 32 + 3), (1, 2 ** 31)])
def test_host_arrays_past_32_bits(shape):
    """Sizes that the library's 32 bits do not hold (memory that is never touched)."""
    with pytest.raises(M.MignonError, match="fewer than 2\\^31"):
        M.token_logprobs(np.zeros(shape, np.float16))

"""The largest sizes of the 8-bit floating-point entry points: refusals, before any launch. CPU only (tests/test_gpu_fp8_limits.py holds
the calls at the limits)."""

import pytest

from vybforge_amd import _lib

A = 1 << 40


@pytest.mark.parametrize("M,K", [(2 ** 28 - 15, 16), (2 ** 28 - 1, 128), (2 ** 27 - 7, 144)])
def test_quantizer_of_too_many_blocks(M, K):
    """2^32 threads, which no launch holds."""
    assert _lib.lib.vybdq_quant_fp8(A, 1, K + 16, 2 * A, 3 * A, M, K, 0) == _lib.ERR_SHAPE
    assert "2^28 - 16" in _lib.last_error()


def test_linear_of_too_many_blocks():
    M, K = 2 ** 24 - 1, 17 * 128
    assert _lib.lib.vybdq_linear_fp8(A, 2 * A, 3 * A, 1, K, 4 * A, M, 1, K, 0, 0, 0, 5 * A, 1 << 39, 0) == _lib.ERR_SHAPE
    assert "2^28 - 16" in _lib.last_error()

"""CPU: sizes and pointers that the sequence operators refuse because a kernel could not take them."""
import pytest

from test_seq_checks import INVALID, P, UNSUPPORTED, call  # noqa: F401


def test_more_columns_than_the_kernels_count():
    """Kernels step past the last column in 32 bits."""
    for cols in ((1 << 30) + 1, (1 << 31) - 1):
        assert call("vdt_quantize_rows", P, 0, 1, cols, cols, P, cols, P, None) == UNSUPPORTED
        assert call("vdt_int8_matmul", P, 32, P, P, 32, P, None, 3, cols, 20, 2, P, cols, None) == UNSUPPORTED
        assert call("vdt_int8_linear", P, 1, 20, P, 32, P, None, 3, cols, 20, 1, P, cols, P, 1 << 20, None) == UNSUPPORTED

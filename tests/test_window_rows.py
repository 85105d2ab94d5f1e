"""Windows and keys' weights take up to 2^31 - 1024 rows: their kernels number the rows of a block, or the one behind, in 31 bits (no kernel
is launched here)."""
import ctypes

import pytest

from simplical_attn_amd import _lib

ONE = ctypes.c_void_p(256)           # never dereferenced: validation fails first


@pytest.mark.parametrize("N", [(1 << 31) - 1, (1 << 31) - 256, (1 << 31) - 1023])
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_rows_close_to_2_to_31(N, dtype):
    _lib.host()
    lib, s = _lib.load(), _lib.stride_array([(1 << 35, 8, 8)] * 8)
    assert lib.sa2_window_forward(ONE, ONE, ONE, ONE, None, ONE, None, 0, 1, N, 1, 1, 8, s, 4, 0, 1.0, dtype, 0, None) == -9
    assert lib.sa2_window_backward(ONE, ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, ONE, ONE, 1 << 62, None, 0, 1, N, 1, 1, 8, s, 4, 0, 1.0, dtype, 0, None) == -9
    assert lib.sa2_window_bwd_workspace_bytes(0, 1, N, 1, 1, 8, 4, 0, dtype, 0) == 0 < lib.sa2_window_bwd_workspace_bytes(0, 1, (1 << 31) - 1024, 1, 1, 8, 4, 0, dtype, 0)
    assert lib.sa2_key_weights(ONE, ONE, ONE, ONE, None, 0, ONE, 1 << 62, None, 0, 1, N, 1, 1, 8, s, 4, 0, 1.0, dtype, 0, None) == -9
    assert lib.sa2_key_weights_workspace_bytes(0, 1, N, 1, 1, 8, 4, 0, dtype, 0) == 0

"""What a windowed backward pass needs beside its tensors (no kernel is launched here)."""
import pytest

from simplical_attn_amd import _lib


@pytest.mark.parametrize("dtype,D", [(0, 64), (1, 128), (2, 128), (1, 256)])
@pytest.mark.parametrize("N,sequences,sinks", [(8192, 512, 128), (32768, 4096, 150), (32768, 1024, 4096), (65536, 512, 65535), (300, 300, 200), (5, 1, 5), (131072, 20, 4), (8192, 0, 4000), (200, 0, 150),
                                               (1 << 20, 1 << 20, 65535)])
def test_first_keys_sums_stay_of_the_tensors_size(N, sequences, sinks, dtype, D):
    """Two fp32 rows at most for each row of dK and of dV, however many sequences share the rows."""
    _lib.host()
    size = lambda s: _lib.load().sa2_window_bwd_workspace_bytes(sequences, 1, N, 16, 8, D, 3, s, dtype, 0)  # noqa: E731
    assert 0 < size(sinks) - size(0) <= 2 * 2 * N * 8 * D * 4 + 256

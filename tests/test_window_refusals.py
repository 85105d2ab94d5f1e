"""What windowed attention, gathered weights and eviction refuse, before anything reaches the GPU (no kernel is launched here)."""
import ctypes

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib

ONE = ctypes.c_void_p(256)           # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    _lib.host()
    return _lib.load()


def t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("kw", [dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(sinks=2)])
@pytest.mark.parametrize("call", [
    lambda **kw: sa.causal_attention(t(1, 5, 4, 8), t(1, 5, 2, 8), t(1, 5, 2, 8), **kw),
    lambda **kw: sa.causal_attention_forward(t(1, 5, 4, 8), t(1, 5, 2, 8), t(1, 5, 2, 8), **kw),
    lambda **kw: sa.causal_attention_backward(t(1, 5, 4, 8), t(1, 5, 2, 8), t(1, 5, 2, 8), t(1, 5, 4, 8), t(1, 4, 5), t(1, 5, 4, 8), **kw)])
def test_windows_of_prompts(lib, call, kw):
    with pytest.raises(ValueError):
        call(**kw)


def test_windows_run_on_the_gpu_only(lib):
    with pytest.raises(RuntimeError, match="GPU only"):
        sa.causal_attention(t(1, 5, 4, 8), t(1, 5, 2, 8), t(1, 5, 2, 8), window=3)
    with pytest.raises(TypeError):
        sa.causal_attention(t(1, 5, 4, 8), t(1, 5, 2, 8), t(1, 5, 2, 8), window="3")


def test_c_entries_of_prompts(lib):
    s = _lib.stride_array([(4096, 64, 8)] * 8)

    def forward(window=4, sinks=1, B=1, N=64, H=4, HK=2, D=8, q=ONE, dtype=0):
        return lib.sa2_window_forward(q, ONE, ONE, ONE, None, ONE, None, 0, B, N, H, HK, D, s, window, sinks, 1.0, dtype, 0, None)

    assert forward(window=0) == forward(window=-1) == forward(sinks=-1) == -5
    assert forward(q=None) == -1 and forward(dtype=9) == -2 and forward(D=257) == -3 and forward(HK=3) == -11
    assert forward(N=1 << 28, H=4, HK=4, sinks=1 << 27) == -9

    def size(window=4, sinks=1, sequences=0, B=1, N=4096, H=4, HK=2, D=64, dtype=1):
        return lib.sa2_window_bwd_workspace_bytes(sequences, B, N, H, HK, D, window, sinks, dtype, 0)

    assert size(window=0) == size(sinks=-1) == size(HK=3) == size(N=0) == 0
    assert size(window=5000, sinks=3) == lib.sa2_causal_bwd_workspace_bytes(1, 4096, 4, 2, 64, 1, 0)
    assert size(sinks=4) > size(sinks=0) > 0 and size(sinks=4, sequences=3) > size(sinks=4)

    def backward(window=4, sinks=1, workspace=ONE, nbytes=1 << 30):
        return lib.sa2_window_backward(ONE, ONE, ONE, ONE, None, ONE, ONE, ONE, ONE, ONE, workspace, nbytes, None, 0, 1, 64, 4, 2, 8, s, window, sinks, 1.0, 0, 0, None)

    assert backward(window=0) == backward(sinks=-2) == -5
    assert backward(workspace=None) == -1 and backward(nbytes=8) == -6

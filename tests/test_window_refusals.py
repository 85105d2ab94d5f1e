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


def _tree(q=(2, 1, 4, 8), k=(2, 1, 2, 8), cache=(6, 16, 2, 8), **kw):
    return sa.tree_attention(t(*q), t(*k), t(*k), None, t(*cache), t(*cache), ints(3, 4), ints(*range(6)).view(2, 3), **kw)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(window=0)), (ValueError, dict(window=2, sinks=-1)), (ValueError, dict(sinks=1)),
    (ValueError, dict(weights=t(2, 2, 47))), (ValueError, dict(weights=t(2, 4, 48))), (ValueError, dict(weights=t(1, 2, 48))), (ValueError, dict(weights=t(2, 48))),
    (ValueError, dict(weights=t(2, 2, 48, dtype=torch.float16))), (ValueError, dict(weights=t(2, 48, 2).transpose(1, 2))),
    (ValueError, dict(weights=t(1, 1, 1).expand(2, 2, 48))),
    (ValueError, dict(q=(2, 3, 4, 8), k=(2, 3, 2, 8), weights=t(2, 2, 48))),
    (RuntimeError, dict(weights=t(2, 2, 48).requires_grad_(True))),
    (RuntimeError, dict(weights=t(2, 2, 48))), (RuntimeError, dict(window=5))])
def test_trees(lib, error, kw):
    with pytest.raises(error):
        _tree(**kw)


def test_inference_tensors_gather_no_weights_outside_of_inference_mode(lib):
    with torch.inference_mode():
        weights = t(2, 2, 48)
    with pytest.raises(RuntimeError, match="inference"):
        _tree(weights=weights)


def test_c_entries_of_trees(lib):
    s = _lib.stride_array([(4096, 64, 8)] * 6 + [(128, 64, 0)])

    def tree(window=4, sinks=1, weights=None, T=1, workspace=ONE, nbytes=1 << 30, strides=s):
        return lib.sa2_window_tree_attention(ONE, ONE, ONE, ONE, ONE, ONE, weights, None, ONE, None, workspace, nbytes, 2, T, 4, 2, 8, 4096, 4, 1, strides, window, sinks, 1.0, 0, 0, None)

    assert tree(window=-1) == tree(sinks=-1) == -5
    assert tree(weights=ONE, T=2) == -14 and tree(T=65) == -14
    assert tree(weights=ONE, nbytes=100) == tree(weights=ONE, workspace=None) == -6
    assert tree(weights=ONE, strides=_lib.stride_array([(4096, 64, 8)] * 6 + [(0, 64, 0)])) == -4

    def size(window=0, sinks=0, weighted=0, T=1, width=64):
        return lib.sa2_window_tree_workspace_bytes(2, T, 4, 2, 64, 64, width, window, sinks, weighted, 1, 0)

    assert size(window=-1) == size(weighted=1, T=2) == 0
    assert size() == lib.sa2_tree_workspace_bytes(2, 1, 4, 2, 64, 64, 64, 1, 0)
    assert size(window=200) < size() < size(weighted=1) and size(window=200, weighted=1) < size(weighted=1)


def _sums(q=(1, 5, 4, 8), k=(1, 5, 2, 8), lse=(1, 4, 5), **kw):
    return sa.key_weights(t(*q), t(*k), lse if isinstance(lse, torch.Tensor) else t(*lse), **kw)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(k=(1, 4, 2, 8))), (ValueError, dict(k=(1, 5, 3, 8))), (ValueError, dict(lse=(1, 5, 4))), (ValueError, dict(lse=t(1, 4, 5, dtype=torch.float64))),
    (ValueError, dict(lse=t(1, 5, 4).transpose(1, 2))), (ValueError, dict(q=(5, 4, 8), k=(5, 2, 8), lse=(4, 5))), (ValueError, dict(window=0)), (ValueError, dict(sinks=2)),
    (ValueError, dict(weights=t(1, 2, 9))), (ValueError, dict(lengths=ints(0))), (ValueError, dict(weights=t(1, 4, 9), lengths=ints(0))),
    (ValueError, dict(weights=t(1, 2, 9), lengths=ints(0, 0))), (ValueError, dict(weights=t(1, 2, 9, dtype=torch.float16), lengths=ints(0))),
    (ValueError, dict(weights=t(1, 9, 2).transpose(1, 2), lengths=ints(0))), (RuntimeError, dict(weights=t(1, 2, 9).requires_grad_(True), lengths=ints(0))),
    (RuntimeError, dict(lse=t(1, 4, 5).requires_grad_(True))), (RuntimeError, dict())])
def test_key_weights(lib, error, kw):
    with pytest.raises(error):
        _sums(**kw)


def _evict(cache=(6, 16, 2, 8), weights=(2, 2, 48), lengths=ints(3, 4), keep=5, table=ints(*range(6)).view(2, 3), **kw):
    make = lambda x: x if isinstance(x, torch.Tensor) else t(*x)  # noqa: E731
    cache = make(cache)
    return sa.cache_evict(cache, cache.clone(), make(weights), lengths, keep, page_table=table, **kw)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(keep=0)), (ValueError, dict(first=-1)), (ValueError, dict(recent=-1)), (ValueError, dict(first=3, recent=3)), (ValueError, dict(keep=1 << 31)),
    (ValueError, dict(weights=(2, 2, 47))), (ValueError, dict(weights=(2, 3, 48))), (ValueError, dict(weights=(3, 2, 48))), (ValueError, dict(weights=(2, 48))),
    (ValueError, dict(weights=t(2, 2, 48, dtype=torch.bfloat16))), (ValueError, dict(weights=t(2, 48, 2).transpose(1, 2))), (ValueError, dict(lengths=ints(1, 2, 3))),
    (ValueError, dict(lengths=ints(1, 2).long())), (ValueError, dict(table=None)), (ValueError, dict(cache=(6, 0, 2, 8))), (ValueError, dict(cache=(6, 16, 2, 264))),
    (TypeError, dict(cache=t(6, 16, 2, 8, dtype=torch.float64))), (RuntimeError, dict(cache=t(6, 16, 2, 8).requires_grad_(True))), (RuntimeError, dict())])
def test_evict(lib, error, kw):
    with pytest.raises(error):
        _evict(**kw)


def test_c_entries_of_weights_and_eviction(lib):
    s = _lib.stride_array([(4096, 64, 8)] * 3)

    def sums(q=ONE, window=0, sinks=0, B=1, N=64, H=4, HK=2, D=8, dtype=0, lengths=None, places=0, workspace=ONE, nbytes=1 << 30, strides=s):
        return lib.sa2_key_weights(q, ONE, ONE, ONE, lengths, places, workspace, nbytes, None, 0, B, N, H, HK, D, strides, window, sinks, 1.0, dtype, 0, None)

    assert sums(q=None) == -1 and sums(dtype=5) == -2 and sums(D=0) == -3 and sums(HK=3) == -11 and sums(window=-1) == sums(window=3, sinks=-1) == -5
    assert sums(lengths=ONE, places=0) == -3 and sums(N=4096, nbytes=4) == -6
    assert sums(B=2, strides=_lib.stride_array([(4096, 64, 8), (4096, 64, 8), (0, 64, 8)])) == -4
    assert lib.sa2_key_weights_workspace_bytes(0, 1, 4096, 4, 2, 64, 0, 0, 1, 0) > 0 == lib.sa2_key_weights_workspace_bytes(0, 1, 4096, 4, 3, 64, 0, 0, 1, 0)

    def evict(k=ONE, B=2, HK=2, heads=2, D=8, page=16, pages=6, width=1, places=16, keep=5, first=0, recent=0, dtype=0, strides=s):
        return lib.sa2_cache_evict(k, ONE, ONE, ONE, ONE, ONE, None, B, HK, heads, D, page, pages, width, places, keep, first, recent, strides, dtype, None)

    assert evict(k=None) == -1 and evict(dtype=7) == -2 and evict(B=0) == evict(D=257) == -3 and evict(heads=3) == -11
    assert evict(page=0) == evict(pages=1) == evict(width=2) == evict(page=(1 << 31) - 64, places=1 << 40) == -13
    assert evict(keep=0) == evict(first=-1) == evict(recent=-1) == evict(first=3, recent=3) == evict(places=15) == -15
    assert evict(strides=_lib.stride_array([(0, 64, 8)] * 3)) == -4


def test_one_cache_twice(lib):
    cache = t(6, 16, 2, 8)
    with pytest.raises(ValueError, match="same memory"):
        sa.cache_evict(cache, cache, t(2, 2, 48), ints(3, 4), 5, page_table=ints(*range(6)).view(2, 3))


def test_first_keys_that_are_too_many(lib):
    s = _lib.stride_array([(1 << 20, 8, 8)] * 3)
    assert lib.sa2_key_weights(ONE, ONE, ONE, ONE, None, 0, ONE, 1 << 40, None, 0, 1, 1 << 17, 1, 1, 8, s, 3, 65536, 1.0, 0, 0, None) == -9
    assert lib.sa2_key_weights_workspace_bytes(0, 1, 1 << 17, 1, 1, 8, 3, 65536, 0, 0) == 0

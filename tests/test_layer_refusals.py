"""What the operators of ordinary attention layers refuse, before anything reaches the GPU (no kernel is launched here)."""
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


F64 = torch.ones(4, dtype=torch.float64)


@pytest.mark.parametrize("error,call", [
    (ValueError, lambda: sa.rotary_embedding(t(2, 8), None, F64)),
    (TypeError, lambda: sa.rotary_embedding(t(1, 2, 3, 8, dtype=torch.float64), None, F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), t(1, 3, 3, 8), F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), t(2, 3, 8), F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), t(1, 2, 3, 8, dtype=torch.float16), F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 6), None, F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 264), None, F64)),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), None, F64.float())),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), None, F64.clone().requires_grad_(True))),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), None, F64, positions=ints(0, 1))),
    (ValueError, lambda: sa.rotary_embedding(t(2, 3, 8), None, F64, positions=t(2))),
    (ValueError, lambda: sa.rotary_embedding(t(2, 3, 8), None, F64, positions=ints(0, 1), cu_seqlens=ints(0, 2))),
    (ValueError, lambda: sa.rotary_embedding(t(1, 2, 3, 8), None, F64, cu_seqlens=ints(0, 2))),
    (ValueError, lambda: sa.rotary_embedding(t(2, 3, 8), None, F64, cu_seqlens=ints(0))),
    (ValueError, lambda: sa.rotary_embedding(t(2, 3, 8), None, F64, cu_seqlens=ints(0, 2).long())),
    (RuntimeError, lambda: sa.rotary_embedding(t(2, 3, 8), None, F64)),
    (ValueError, lambda: sa.rotary_frequencies(7)),
    (ValueError, lambda: sa.rotary_frequencies(8, scaling="other")),
    (ValueError, lambda: sa.rotary_frequencies(8, scaling="parts", factor=2.0)),
    (ValueError, lambda: sa.rotary_frequencies(2, scaling="base", factor=2.0)),
    (ValueError, lambda: sa.rotary_frequencies(8, factor=0.0)),
])
def test_rotary(lib, error, call):
    with pytest.raises(error):
        call()


def _append(k=(2, 3, 2, 8), v=None, kc=(4, 16, 2, 8), vc=None, lengths=ints(0, 0), table=ints(0, 1, 2, 3).view(2, 2), **kw):
    v, vc = v or k, vc or kc
    make = lambda x: x if isinstance(x, torch.Tensor) else t(*x)
    return sa.cache_append(make(k), make(v), make(kc), make(vc), lengths, table, **kw)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(k=(3, 8))),
    (ValueError, dict(v=(2, 3, 1, 8))),
    (ValueError, dict(kc=(4, 16, 1, 8))),
    (ValueError, dict(kc=(4, 16, 2, 16))),
    (ValueError, dict(vc=(4, 8, 2, 8))),
    (ValueError, dict(kc=(4, 0, 2, 8))),
    (ValueError, dict(kc=t(4, 16, 8, 2).transpose(2, 3))),
    (ValueError, dict(kc=t(4, 16, 2, 8, dtype=torch.float16))),
    (ValueError, dict(lengths=ints(0))),
    (ValueError, dict(lengths=ints(0, 0).long())),
    (ValueError, dict(table=ints(0, 1))),
    (ValueError, dict(table=ints(0, 1).view(1, 2))),
    (ValueError, dict(table=None)),
    (ValueError, dict(rows=ints(0, 1))),
    (ValueError, dict(rows=ints(0, 1).view(1, 2))),
    (ValueError, dict(k=(5, 2, 8))),
    (ValueError, dict(k=(5, 2, 8), cu_seqlens=ints(0, 2, 5), rows=ints(0, 0).view(2, 1))),
    (ValueError, dict(k=(2, 3, 2, 264), kc=(4, 16, 2, 264))),
    (RuntimeError, dict(k=t(2, 3, 2, 8).requires_grad_(True))),
    (RuntimeError, dict()),
])
def test_append(lib, error, kw):
    with pytest.raises(error):
        _append(**kw)


@pytest.mark.parametrize("error,call", [
    (ValueError, lambda: sa.causal_attention(t(2, 8), t(2, 8), t(2, 8))),
    (TypeError, lambda: sa.causal_attention(*[t(1, 2, 3, 8, dtype=torch.int32)] * 3)),
    (ValueError, lambda: sa.causal_attention(t(1, 2, 4, 8), t(1, 3, 4, 8), t(1, 2, 4, 8))),
    (ValueError, lambda: sa.causal_attention(t(1, 2, 4, 8), t(1, 2, 4, 8), t(1, 2, 2, 8))),
    (ValueError, lambda: sa.causal_attention(t(1, 2, 4, 8), t(1, 2, 3, 8), t(1, 2, 3, 8))),
    (ValueError, lambda: sa.causal_attention(t(1, 2, 4, 8), t(1, 2, 4, 8), t(1, 2, 4, 8, dtype=torch.float16))),
    (ValueError, lambda: sa.causal_attention(*[t(1, 2, 4, 257)] * 3)),
    (ValueError, lambda: sa.causal_attention(*[t(5, 4, 8)] * 3)),
    (ValueError, lambda: sa.causal_attention(*[t(1, 5, 4, 8)] * 3, cu_seqlens=ints(0, 5))),
    (ValueError, lambda: sa.causal_attention(*[t(5, 4, 8)] * 3, cu_seqlens=ints(0, 5).long())),
    (RuntimeError, lambda: sa.causal_attention(*[t(5, 4, 8)] * 3, cu_seqlens=ints(0, 5))),
    (ValueError, lambda: sa.causal_attention_backward(*[t(1, 5, 4, 8)] * 3, t(1, 5, 4, 8), t(1, 4, 5), t(1, 5, 4, 8), needs=(True,))),
])
def test_causal(lib, error, call):
    with pytest.raises(error):
        call()


def _tree(q=(2, 3, 4, 8), k=(2, 3, 2, 8), parents=ints(-1, 0, 1, -1, -1, 0).view(2, 3), kc=(4, 16, 2, 8), lengths=ints(0, 0),
          table=ints(0, 1, 2, 3).view(2, 2), v=None):
    make = lambda x: x if isinstance(x, torch.Tensor) else t(*x)
    return sa.tree_attention(make(q), make(k), make(v or k), parents, make(kc), make(kc), lengths, table)


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(q=(6, 4, 8))),
    (ValueError, dict(q=(2, 65, 4, 8), k=(2, 65, 2, 8), parents=None)),
    (ValueError, dict(q=(2, 0, 4, 8), k=(2, 0, 2, 8), parents=None)),
    (ValueError, dict(q=(2, 3, 3, 8))),
    (ValueError, dict(v=(2, 3, 4, 8))),
    (ValueError, dict(q=(2, 3, 4, 260), k=(2, 3, 2, 260), kc=(4, 16, 2, 260))),
    (ValueError, dict(parents=ints(-1, 0, 1))),
    (ValueError, dict(parents=ints(-1, 0).view(1, 2))),
    (ValueError, dict(parents=ints(-1, 0, 1, -1, -1, 0).view(2, 3).long())),
    (ValueError, dict(kc=(4, 16, 4, 8))),
    (ValueError, dict(table=None)),
    (ValueError, dict(lengths=ints(0, 0, 0))),
    (RuntimeError, dict(q=t(2, 3, 4, 8).requires_grad_(True))),
    (RuntimeError, dict()),
])
def test_tree(lib, error, kw):
    with pytest.raises(error):
        _tree(**kw)


def test_c_abi(lib):
    st = _lib.stride_array([(1024, 128, 64)] * 4)

    def rotary(q=ONE, k=ONE, f=ONE, pos=None, bytes_=0, cu=None, seqs=0, B=1, N=8, H=2, HK=2, D=64, rot=64, strides=st, dtype=0):
        return lib.sa2_rotary(q, k, ONE, ONE, f, pos, bytes_, cu, seqs, B, N, H, HK, D, rot, strides, 1.0, 0, 0, dtype, None)

    assert rotary(q=None) == -1 and rotary(k=None) == -1 and rotary(f=None) == -1
    assert rotary(dtype=3) == -2
    assert rotary(B=0) == -3 and rotary(D=257) == -3 and rotary(HK=-1) == -3 and rotary(cu=ONE, seqs=0) == -3 and rotary(B=2, cu=ONE, seqs=1) == -3
    assert rotary(rot=63) == -12 and rotary(rot=66) == -12 and rotary(rot=0) == -12 and rotary(pos=ONE, bytes_=2) == -12
    assert rotary(N=1 << 30, H=2) == -9
    assert rotary(strides=_lib.stride_array([(1024, 0, 64)] * 4)) == -4

    def append(k=ONE, lengths=ONE, table=ONE, rows=None, nrows=0, cu=None, seqs=0, B=2, N=8, HK=2, D=64, page=16, pages=4, width=2, strides=st, dtype=0):
        return lib.sa2_cache_append(k, ONE, ONE, ONE, lengths, table, rows, nrows, cu, seqs, B, N, HK, D, page, pages, width, strides, dtype, None)

    assert append(k=None) == -1 and append(lengths=None) == -1
    assert append(dtype=9) == -2
    assert append(N=0) == -3 and append(rows=ONE) == -3 and append(rows=ONE, nrows=2, B=1, cu=ONE, seqs=2) == -3
    assert append(page=0) == -13 and append(pages=0) == -13 and append(width=0) == -13 and append(table=None, pages=1) == -13
    assert append(strides=_lib.stride_array([(1024, 0, 64)] * 4)) == -4

    st = _lib.stride_array([(1024, 128, 64)] * 8)

    def causal(q=ONE, cu=None, seqs=0, B=1, N=8, H=2, HK=2, D=64, strides=st, dtype=1):
        return lib.sa2_causal_forward(q, ONE, ONE, ONE, None, ONE, cu, seqs, B, N, H, HK, D, strides, 0.1, dtype, 0, None)

    assert causal(q=None) == -1 and causal(dtype=5) == -2 and causal(N=0) == -3 and causal(D=257) == -3 and causal(B=2, cu=ONE, seqs=3) == -3
    assert causal(HK=3) == -11 and causal(HK=0) == -11 and causal(N=1 << 30) == -9
    assert causal(strides=_lib.stride_array([(1024, 128, 0)] * 8)) == -4
    need = lib.sa2_causal_bwd_workspace_bytes(1, 8, 2, 2, 64, 1, 0)
    assert need >= 2 * 8 * 4 and lib.sa2_causal_bwd_workspace_bytes(1, 8, 3, 2, 64, 1, 0) == 0

    def backward(workspace=ONE, size=need, dq=ONE, H=2):
        return lib.sa2_causal_backward(ONE, ONE, ONE, ONE, None, ONE, ONE, dq, None, None, workspace, size, None, 0, 1, 8, H, 2, 64, st, 0.1, 1, 0, None)

    assert backward(workspace=None) == -1 and backward(size=need - 1) == -6 and backward(workspace=ctypes.c_void_p(264)) == -6 and backward(H=3) == -11
    assert backward(dq=None) == 0                         # no gradient is wanted: nothing is launched

    def tree(q=ONE, lengths=ONE, table=ONE, B=2, T=4, H=4, HK=2, D=64, page=16, pages=4, width=2, strides=st, dtype=1):
        return lib.sa2_tree_attention(q, ONE, ONE, ONE, ONE, ONE, None, lengths, table, None, 0, B, T, H, HK, D, page, pages, width, strides, 0.1, dtype, 0, None)

    assert tree(q=None) == -1 and tree(lengths=None) == -1 and tree(dtype=-1) == -2 and tree(B=0) == -3
    assert tree(HK=3) == -11 and tree(T=65) == -14 and tree(page=0) == -13 and tree(pages=0) == -13 and tree(table=None) == -13
    assert tree(table=None, pages=1, width=1) == -13 and tree(page=1 << 20, width=1 << 12) == -13
    assert tree(strides=_lib.stride_array([(1024, -1, 64)] * 8)) == -4
    assert lib.sa2_tree_workspace_bytes(1, 1, 8, 2, 128, 64, 512, 1, 0) > 0 and tree(page=64, pages=512, width=512) == -6
    assert lib.sa2_tree_workspace_bytes(1, 65, 8, 2, 128, 64, 512, 1, 0) == 0
    seen = {lib.sa2_strerror(code) for code in range(-14, 0)}
    assert len(seen) == 14 and not any(b"unknown sa2" in m for m in seen)

"""Causal attention and large drafted trees where a row's first 32 keys say little about the others: values so large that weights above
1 take the sums out of fp32's range, first keys whose scores are minus infinity, fp16 weights below 2^-25 of the largest."""
import math

import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16 = torch.bfloat16, torch.float16
E = 2.0 ** -24


def _rows(heads, N, D, dtype, seed):
    """q [1, N, heads, D], k, v [1, N, 1, D]; scores of scale 1 / 8: column 0 of q is 8, so that column 0 of k is added to them."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(1, N, h, D, generator=g).to(DEV) for h in (heads, 1, 1))
    q[..., 0] = 8
    k[..., 0] = 0
    return [x.to(dtype) for x in (q, k, v)]


def _check(out, q, k, v, rows, scale, seen=None):
    """Bounds as in causal_util.py, of rows `rows` of one sequence (seen: their masks, else causal)."""
    t = torch.finfo(out.dtype).eps / 2
    Q, K, V, D = q[rows].double(), k.double(), v.double(), q.shape[-1]
    n = len(K)
    M = seen if seen is not None else torch.arange(n, device=DEV)[None] <= torch.arange(n, device=DEV)[rows, None]
    S = (Q @ K.T * scale).masked_fill(~M, -math.inf)
    P = torch.softmax(S, 1)
    r = ((D + 4) * E * scale * (Q.abs() @ K.abs().nan_to_num(posinf=0).T)).masked_fill(~M, 0).amax(1, keepdim=True)
    want = P @ V
    # fp16: of the keys up to the row's own at most 2^-25 each, less by the power of two that their number brings (2^15: 1, up to 2^8)
    keys = M.sum(1, keepdim=True).double().clamp(min=1)
    low = 2.0 ** (-25 - (keys.log2().ceil() - 14).clamp(0, 8)) if out.dtype == FP16 else 0.0
    bound = (P @ V.abs()) * (2 * r + t + (n + 16) * E) + low * (M.double() @ V.abs()) + t * want.abs() + 2.0 ** -24
    x = out[rows].double()
    assert torch.isfinite(x).all()
    assert ((x - want).abs() <= bound).all()


@pytest.mark.parametrize("size", [90, 120])
@pytest.mark.parametrize("rise", [3.0, 8.0, 40.0])
@pytest.mark.parametrize("heads,D", [(2, 64), (2, 128), (192, 64), (192, 128)])
def test_large_values(heads, D, rise, size):
    """bf16 values of 2^size and keys from the 300th on with scores `rise` above the first ones'."""
    q, k, v = _rows(heads, 700, D, BF16, D)
    k[:, 300:, :, 0] = rise
    v = (v.double().clamp(-4, 4) * 2.0 ** size).to(BF16)
    out = sa.causal_attention(q, k, v, scale=0.125)
    # (with weights of at most 1, 700 values of up to 2^122 are in range)
    for h in (0, heads - 1):
        _check(out[0, :, h], q[0, :, h], k[0, :, 0], v[0, :, 0], slice(None), 0.125)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads,D", [(2, 64), (2, 128), (192, 128)])
def test_first_keys_without_a_score(heads, D, dtype):
    """The first 32 keys' scores are minus infinity, the others' far below zero."""
    q, k, v = _rows(heads, 600, D, dtype, D + 1)
    k[..., 0] = -300
    k[:, :32, :, 0] = -math.inf
    out = sa.causal_attention(q, k, v, scale=0.125)
    for h in (0, heads - 1):
        _check(out[0, :, h], q[0, :, h], k[0, :, 0], v[0, :, 0], slice(32, None), 0.125)


def _tree(q, k, v, T, **kw):
    """The last T rows of q as a chain of drafted nodes over the other rows of k and v."""
    n = k.shape[1] - T
    cut = lambda x, a, b: x[:, a:b].contiguous()
    lengths = torch.tensor([n], dtype=torch.int32, device=DEV)
    return sa.tree_attention(cut(q, n, n + T), cut(k, n, n + T), cut(v, n, n + T), None, cut(k, 0, n), cut(v, 0, n), lengths, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rise", [8.0, 40.0])
@pytest.mark.parametrize("size", [100, 120])
def test_large_values_in_trees(D, rise, size):
    q, k, v = _rows(4, 40 + 3000, D, BF16, D + 2)
    k[:, 200:, :, 0] = rise
    v = (v.double().clamp(-4, 4) * 2.0 ** size).to(BF16)
    out = _tree(q, k, v, 40, scale=0.125)
    for h in (0, 3):
        _check(torch.cat((out[0, :1, h].expand(3000, D), out[0, :, h])), q[0, :, h], k[0, :, 0], v[0, :, 0], slice(3000, None), 0.125)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_first_keys_without_a_score_in_trees(dtype):
    q, k, v = _rows(4, 40 + 2000, 128, dtype, 4)
    k[..., 0] = -300
    k[:, :700, :, 0] = -math.inf
    out = _tree(q, k, v, 40, scale=0.125)
    for h in (0, 3):
        _check(torch.cat((out[0, :1, h].expand(2000, 128), out[0, :, h])), q[0, :, h], k[0, :, 0], v[0, :, 0], slice(2000, None), 0.125)


@pytest.mark.parametrize("T", [1, 12, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_a_cached_key_far_above_all_others(D, T):
    """fp16: the first key's weight is 2^25 times every other one's, whose sum still counts."""
    N = 40000
    g = torch.Generator().manual_seed(D)
    v = 32 * (torch.randn(1, N + T, 1, D, generator=g).to(DEV).half().abs() + 1)
    v[:, 0] = -0.01
    k = torch.zeros(1, N + T, 1, D, dtype=FP16, device=DEV)
    q = torch.zeros(1, N + T, 4, D, dtype=FP16, device=DEV)
    q[..., 0], k[:, 0, :, 0] = 1, 17.5
    out = _tree(q, k, v, T, scale=1.0)
    for h in (0, 3):
        _check(torch.cat((out[0, :1, h].expand(N, D), out[0, :, h])), q[0, :, h], k[0, :, 0], v[0, :, 0], slice(N, None), 1.0)


def test_a_key_far_above_all_others():
    """fp16: the first key's weight is 2^25 times every other one's, whose sum still counts."""
    N, D = 24000, 64
    g = torch.Generator().manual_seed(33)
    v = 32 * (torch.randn(1, N, 1, D, generator=g).to(DEV).half().abs() + 1)
    v[:, 0] = -0.01
    k = torch.zeros(1, N, 1, D, dtype=FP16, device=DEV)
    q = torch.zeros(1, N, 2, D, dtype=FP16, device=DEV)
    q[..., 0], k[:, 0, :, 0] = 1, 17.5
    out, lse = sa.causal_attention_forward(q, k, v, scale=1.0)
    for h in (0, 1):
        rows = slice(N - 2000, None, 7)
        _check(out[0, :, h], q[0, :, h], k[0, :, 0], v[0, :, 0], rows, 1.0)
        n = torch.arange(N, device=DEV).double()
        # the score is exact; a logarithm and a product in 32 bits, sums of n terms
        assert ((lse[0, h].double() - (math.exp(17.5) + n).log()).abs() <= (n + 64) * E).all()

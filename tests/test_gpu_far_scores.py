"""Scores very far from zero, as rows of the type's lowest value leave them: queries whose keys are all that low attend to them evenly, others
not at all; keys as far above all others get everything.  Prompts, with a window and without, and trees over a cache, with the weights that they gather."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from tests.window_util import sees

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def _far(dtype, size):
    """(query's column, key's column): their product is `size` of what the type allows."""
    if dtype == FP16:
        return (65504.0, 65504.0) if size else (4096.0, 65504.0)
    return 1.0, (torch.finfo(torch.bfloat16).max, 1e26, 1e34)[size]


def _tensors(lead, heads, D, dtype, g):
    return [torch.randn(*lead, h, D, generator=g).to(dtype).to(DEV) for h in heads]


def _check(out, lse, Q, K, V, visible, scale, dtype, rounded):
    """One head.  Scores of far keys are exact here, and equal to each other; the others are off by r, and as in window_util.py from there on."""
    t = torch.finfo(dtype).eps / 2
    S = (Q.double() @ K.double().T * scale).masked_fill(~visible, -math.inf)
    P = torch.softmax(S, 1)
    n = int(visible.sum(1).max())
    near = K.double().clone()
    near[:, 0] = 0
    r = (K.shape[1] + 4) * E * abs(scale) * (Q.double()[:, 1:].abs() @ near[:, 1:].abs().T).amax(1, keepdim=True)
    rel = 2 * r + (t if rounded else E) + (n + 16) * E
    want = P @ V.double()
    low = 2.0 ** -25 * (visible.double() @ V.double().abs()) if rounded and dtype == FP16 else 0.0
    assert torch.isfinite(out).all()
    far = (out.double() - want).abs() / ((P @ V.double().abs()) * rel + low + t * want.abs() + torch.finfo(dtype).smallest_normal)
    assert far.max() <= 1, far.max().item()
    if lse is not None:
        L = torch.logsumexp(S, 1)
        assert ((lse.double() - L).abs() <= r[:, 0] + (n + 16) * E + 4 * E * L.abs()).all()
    return P, rel


@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 0), (100, 5), (7, 130)])
@pytest.mark.parametrize("B,N,D", [(1, 300, 64), (70, 520, 128), (2, 300, 136), (90, 400, 64), (1, 700, 128)])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("size", [0, 1, 2])
def test_prompts(B, N, D, window, sinks, dtype, size):
    if size == 2 and dtype == FP16:
        pytest.skip("the same")
    g = torch.Generator().manual_seed(N + D)
    q, k, v = _tensors((B, N), (4, 1, 1), D, dtype, g)
    a, b = _far(dtype, size)
    q[..., 0], k[..., 0] = a, 0.0
    k[:, :120] = 0.0                                        # (a sequence's first queries see nothing else)
    k[:, :120, :, 0] = -b
    k[:, 200:260] = 0.0
    k[:, 200:260, :, 0] = -b
    k[:, 280:282] = 0.0
    k[:, 280:282, :, 0] = b
    out, lse = sa.causal_attention_forward(q, k, v, window=window, sinks=sinks)
    visible = sees(N, window or N, sinks, DEV)
    for i in {0, B - 1}:
        for h in (0, 3):
            _check(out[i, :, h], lse[i, h], q[i, :, h], k[i, :, 0], v[i, :, 0], visible, D ** -0.5, dtype, dtype != FP32 and D <= 128)


@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 2), (90, 2), (1400, 2), (300, 100)])
@pytest.mark.parametrize("T,H", [(1, 4), (5, 4), (12, 4), (40, 4), (1, 70)])
@pytest.mark.parametrize("dtype,D", [(BF16, 64), (FP16, 128), (FP32, 64), (BF16, 136)])
@pytest.mark.parametrize("size", [0, 1])
def test_trees(T, H, dtype, D, window, sinks, size):
    g = torch.Generator().manual_seed(T + D)
    rows, held = 1600, (1600, 1333)
    q, k, v = _tensors((2, T), (H, 1, 1), D, dtype, g)
    kc, vc = _tensors((2, rows), (1, 1), D, dtype, g)
    a, b = _far(dtype, size)
    q[..., 0], k[...], kc[..., 0] = a, 0.0, 0.0
    k[..., 0] = -b
    kc[0] = 0.0
    kc[0, ..., 0] = -b                                      # the first sequence has only low rows, the second such ones at its end
    kc[1, 1250:] = 0.0
    kc[1, 1250:, :, 0] = -b
    kc[1, 300:700] = 0.0                                    # (and in tiles before and behind others)
    kc[1, 300:700, :, 0] = -b
    weights = torch.zeros(2, 1, rows, device=DEV) if T == 1 else None
    out = sa.tree_attention(q, k, v, None, kc, vc, torch.tensor(held, dtype=torch.int32, device=DEV), window=window, sinks=sinks, weights=weights)
    for i, n in enumerate(held):
        K, V = (torch.cat((c[i, :n, 0], x[i, :, 0])) for c, x in ((kc, k), (vc, v)))
        visible = sees(n + T, window or n + T, sinks, DEV)[n:]
        sums = off = 0.0
        for h in range(H):
            P, rel = _check(out[i, :, h], None, q[i, :, h], K, V, visible, D ** -0.5, dtype, dtype != FP32 and D <= 128)
            sums, off = sums + P[0], off + P[0] * rel[0]
        if weights is not None:
            places = min(n + 1, rows)
            assert ((weights[i, 0, :places].double() - sums[:places]).abs() <= off[:places] + (H + 2) * E * sums[:places] + 2.0 ** -126).all()
            assert weights[i, 0, places:].count_nonzero() == 0

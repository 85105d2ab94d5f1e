"""key_weights against the definition in 64 bits: types, head layouts, lengths from one on, packed sequences, windows, views,
rows that must not count, sums that go to a cache's places, graphs."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib
from tests.window_util import sees

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def _inputs(lead, H, HK, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*lead, h, D, generator=g) * std).to(dtype).to(DEV) for h in (H, HK)]


def _exact(q, k, lse, scale, window, sinks):
    """One sequence: q [n, G, D], k [n, D], lse [G, n]; (sums, bound).  Scores are off by (D + 4) e scale sum |q||k|, exponents by
    3 e (|score| + |lse|) more (conversion to powers of two), exponentials by 2 e; sums by a term's e for each addition."""
    n, G, D = q.shape
    mask = sees(n, window or n, sinks, q.device)
    sums, off = torch.zeros(n, dtype=torch.float64, device=q.device), torch.zeros(n, dtype=torch.float64, device=q.device)
    for g in range(G):
        Q, K = q[:, g].double(), k.double()
        S = Q @ K.T * scale
        x = (S - lse[g, :, None].double()).masked_fill(~mask, -math.inf)
        P = x.exp()
        r = (D + 4) * E * abs(scale) * (Q.abs() @ K.abs().T) + 3 * E * (S.abs() + lse[g, :, None].double().abs()) + 2 * E
        sums += P.sum(0)
        off += (P * r.masked_fill(~mask, 0)).sum(0)
    most = int(mask.sum(0).max()) * G
    return sums, off + (most + 16) * E * sums + 2.0 ** -126 * most


def _check(got, want):
    far = (got.double() - want[0]).abs() / want[1]
    assert far.max() <= 1, far.max().item()


def _lse(q, k, cu=None, window=None, sinks=0, scale=None):
    return sa.causal_attention_forward(q, k, torch.zeros_like(k), cu, scale, window=window, sinks=sinks)[1]


SHAPES = [(1, 1, 1, 1, 64, None, 0), (2, 3, 2, 1, 64, None, 0), (1, 33, 4, 2, 128, None, 0), (2, 130, 3, 3, 32, None, 0), (1, 257, 8, 1, 128, 40, 0),
          (1, 700, 4, 2, 80, 128, 4), (2, 1100, 8, 2, 128, None, 0), (1, 1500, 16, 4, 64, 300, 70), (1, 300, 2, 1, 256, None, 0), (1, 90, 2, 2, 33, 1, 0),
          (1, 200, 1, 1, 161, 9, 2), (1, 2600, 2, 1, 128, None, 0), (1, 513, 5, 1, 96, 512, 3), (1, 70, 2, 1, 8, None, 0)]


@pytest.mark.parametrize("dtype,flags", [(BF16, 0), (FP16, 0), (FP32, 0), (BF16, _lib.FLAG_FORCE_GENERIC)])
@pytest.mark.parametrize("B,N,H,HK,D,window,sinks", SHAPES)
def test_batches(B, N, H, HK, D, window, sinks, dtype, flags):
    q, k = _inputs((B, N), H, HK, D, dtype, B + N + D)
    lse = _lse(q, k, None, window, sinks)
    got = sa.key_weights(q, k, lse, window=window, sinks=sinks, flags=flags)
    assert got.shape == (B, HK, N) and got.dtype == FP32
    for b in range(B):
        for hk in range(HK):
            hs = slice(hk * (H // HK), (hk + 1) * (H // HK))
            _check(got[b, hk], _exact(q[b, :, hs], k[b, :, hk], lse[b, hs], D ** -0.5, window, sinks))
    # every query's weights are one
    assert ((got.sum(2) - N * H // HK).abs() <= 1e-5 * N * H).all()


@pytest.mark.parametrize("dtype,H,HK,D", [(BF16, 4, 1, 128), (FP16, 2, 1, 64), (FP32, 3, 3, 64), (BF16, 2, 2, 40), (FP32, 1, 1, 200)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (150, 70)])
@pytest.mark.parametrize("ends", [[0, 5], [0, 1, 2, 3], [0, 0, 64, 64, 65, 200], [3, 40, 40, 168, 297], [0, 300, 301, 900], [0, 1030, 1031, 1600]])
def test_packed(ends, dtype, H, HK, D, window, sinks):
    T = ends[-1] + 9
    q, k = _inputs((T,), H, HK, D, dtype, T + D)
    for x in (q, k):                                        # rows of no sequence hold anything
        x[:ends[0]] = math.nan
        x[ends[-1]:] = math.inf
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    lse = _lse(q, k, cu, window, sinks)
    got = sa.key_weights(q, k, lse, cu, window=window, sinks=sinks)
    assert got.shape == (HK, T) and got[:, :ends[0]].count_nonzero() == 0 and got[:, ends[-1]:].count_nonzero() == 0
    places = torch.rand(len(ends) - 1, HK, 700, generator=torch.Generator().manual_seed(1)).to(DEV)
    held = torch.tensor([(37 * i) % 90 for i in range(len(ends) - 1)], dtype=torch.int32, device=DEV)
    held[0] = 690
    before = places.clone()
    assert sa.key_weights(q, k, lse, cu, window=window, sinks=sinks, weights=places, lengths=held) is None
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        for hk in range(HK):
            hs = slice(hk * (H // HK), (hk + 1) * (H // HK))
            if b > a:
                _check(got[hk, a:b], _exact(q[a:b, hs], k[a:b, hk], lse[hs, a:b], D ** -0.5, window, sinks))
            want, n = before[i, hk].clone(), int(held[i])
            taken = got[hk, a:b][:max(0, 700 - n)]
            want[n:n + len(taken)] += taken
            assert torch.equal(places[i, hk], want)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_hidden_queries_may_hold_anything(dtype):
    """A query that a key is hidden from, whatever it holds, adds nothing to it."""
    N, window, at = 400, 60, 200
    q, k = _inputs((1, N), 4, 2, 64, dtype, 3)
    lse = _lse(q, k, None, window, 2)
    want = sa.key_weights(q, k, lse, window=window, sinks=2)
    hidden = ~sees(N, window, 2)[at].to(DEV)
    for bad in (math.nan, math.inf, -math.inf):
        q2, lse2 = q.clone(), lse.clone()
        q2[:, at, :, 3], lse2[..., at] = bad, bad
        got = sa.key_weights(q2, k, lse2, window=window, sinks=2)
        assert torch.equal(got[..., hidden], want[..., hidden])
    k2 = k.clone()
    k2[:, at] = math.nan                                    # a key by itself
    got = sa.key_weights(q, k2, lse, window=window, sinks=2)
    others = torch.arange(N, device=DEV) != at
    assert torch.equal(got[..., others], want[..., others]) and got[..., at].isnan().all()


def test_views_scales_streams_and_graphs():
    g = torch.Generator().manual_seed(9)
    fused = torch.randn(2, 300, 4 + 2 * 2, 65, generator=g).to(BF16).to(DEV)
    for off in (0, 1):                                      # (off the grid of 16 bytes, too)
        q, k = fused[:, :, :4, off:off + 64], fused[:, :, 4:6, off:off + 64]
        for scale in (None, -0.2, 0.0):
            lse = _lse(q.contiguous(), k.contiguous(), scale=scale)
            got = sa.key_weights(q, k, lse, scale=scale)
            for hk in range(2):
                _check(got[1, hk], _exact(q[1, :, 2 * hk:2 * hk + 2], k[1, :, hk], lse[1, 2 * hk:2 * hk + 2], 64 ** -0.5 if scale is None else scale, None, 0))
    q, k = _inputs((2, 900), 8, 2, 128, BF16, 5)
    lse = _lse(q, k)
    want = sa.key_weights(q, k, lse)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sa.key_weights(q, k, lse)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sa.key_weights(q, k, lse)
    for seed in (1, 2, 3):
        q2, k2 = _inputs((2, 900), 8, 2, 128, BF16, seed)
        q.copy_(q2), k.copy_(k2)
        lse.copy_(_lse(q, k))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, sa.key_weights(q, k, lse))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("sinks", [1, 128, 257, 600])
@pytest.mark.parametrize("ends,add", [([0, 700, 700, 1100, 1101, 2000], False), ([0, 700, 700, 1100, 1101, 2000], True), ([5 * i for i in range(101)], True)])
def test_many_first_keys(ends, add, sinks, dtype):
    """Blocks of first keys, whose streams are cut by themselves: of sequences shorter than a block, than the first keys, and longer."""
    H, HK, D, window = 4, 2, 64, 33
    T = ends[-1] + 3
    q, k = _inputs((T,), H, HK, D, dtype, sinks)
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    lse = _lse(q, k, cu, window, sinks)
    got = sa.key_weights(q, k, lse, cu, window=window, sinks=sinks)
    if add:
        places = torch.zeros(len(ends) - 1, HK, 1000, device=DEV)
        sa.key_weights(q, k, lse, cu, window=window, sinks=sinks, weights=places, lengths=torch.zeros(len(ends) - 1, dtype=torch.int32, device=DEV))
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        for hk in range(HK):
            hs = slice(2 * hk, 2 * hk + 2)
            if b > a:
                _check(got[hk, a:b], _exact(q[a:b, hs], k[a:b, hk], lse[hs, a:b], D ** -0.5, window, sinks))
            if add:
                assert torch.equal(places[i, hk, :b - a], got[hk, a:b]) and places[i, hk, b - a:].count_nonzero() == 0
    assert got[:, ends[-1]:].count_nonzero() == 0


def test_bounds_out_of_order():
    """No defined sums, but no access outside of the tensors either: what stands around the places stays."""
    q, k = _inputs((400,), 2, 1, 64, BF16, 3)
    for ends in ([0, 100, 200, 50], [-7, 500, 300, 90], [300, 200, 100, 0], [0, 399, 10, 380]):
        cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
        for window, sinks in ((None, 0), (20, 3)):
            lse = torch.zeros(2, 400, device=DEV)
            wide = torch.full((9, 1, 128), -1.0, device=DEV)
            held = torch.zeros(9, dtype=torch.int32, device=DEV)
            sa.key_weights(q, k, lse, cu, window=window, sinks=sinks, weights=wide[3:6], lengths=held[3:6])
            assert (wide[:3] == -1).all() and (wide[6:] == -1).all()

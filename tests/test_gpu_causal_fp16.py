"""Causal attention in fp16 where its narrow range shows: values far from 1, rows and sequences whose gradients differ by many powers of
two, weights far below a row's largest.  Bounds: causal_fp16_util.py."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from tests.causal_fp16_util import exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FP16 = torch.float16


def _inputs(N, H, HK, D, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(N, h, D, generator=g, dtype=torch.float64).to(DEV) * s for h, s in ((H, std), (HK, std), (HK, 1.0), (H, 1.0))]


def _train(q, k, v, dout, cu, scale=None):
    leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
    out = sa.causal_attention(*leaves, cu, scale)
    return (out.detach(), *torch.autograd.grad(out, leaves, dout))


def _compare(q, k, v, dout, got, ends, names=("out", "dq", "dk", "dv"), scale=None):
    H, HK, D = q.shape[1], k.shape[1], q.shape[2]
    G = H // HK
    for lo, hi in zip(ends, ends[1:]):
        for hk in range(HK):
            hs = slice(hk * G, hk * G + G)
            want = exact(q[lo:hi, hs], k[lo:hi, hk], v[lo:hi, hk], dout[lo:hi, hs], scale or D ** -0.5)
            for name, x in zip(("out", "dq", "dk", "dv"), got):
                if name in names:
                    part = x[lo:hi, hs] if name in ("out", "dq") else x[lo:hi, hk]
                    value, bound = want[name]
                    # (what fp16 cannot hold is an infinity)
                    fits = value.abs() + bound < 65504
                    far = ((part.double() - value).abs() / bound).masked_fill(~fits, 0)
                    assert torch.isfinite(part[fits]).all() and far.max() <= 1, "%s of rows %d..%d: %.3g of its bound off" % (name, lo, hi, far.nan_to_num(math.inf).max())


def _half(*xs):
    return [x.half() for x in xs]


# (the last: enough blocks of 256 queries that a wavefront owns 64)
SIZES = [(2, 1, 1, 64), (150, 2, 1, 128), (333, 4, 2, 64), (700, 2, 2, 80), (1500, 4, 1, 128), (1030, 128, 4, 64), (900, 160, 8, 128)]


@pytest.mark.parametrize("offset", [0.0, 3000.0, 20000.0])
@pytest.mark.parametrize("N,H,HK,D", SIZES)
def test_large_values(N, H, HK, D, offset):
    """Rows of values of 1000 with one sign, or with a common offset: dS exceeds fp16's largest number unless its factor knows of them."""
    q, k, v, dout = _inputs(N, H, HK, D, N + D)
    sign = v[:, :, :1].sign()
    v, dout = (1000 * sign.expand_as(v), torch.full_like(dout, 0.01)) if offset == 0 else (v * 100 + offset * sign, dout * 0.01)
    q, k, v, dout = _half(q, k, v, dout)
    cu = torch.tensor([0, N], dtype=torch.int32, device=DEV)
    _compare(q, k, v, dout, _train(q, k, v, dout, cu), [0, N])


@pytest.mark.parametrize("apart", [12, 15])
@pytest.mark.parametrize("H,HK,D", [(2, 1, 64), (4, 2, 128), (96, 8, 64)])
def test_sequences_of_different_weight(H, HK, D, apart):
    """dO of one sequence, and of the heads of another, 2^apart above the rest."""
    ends = [0, 300, 301, 620, 1000]
    q, k, v, dout = _inputs(1000, H, HK, D, H + D)
    dout[301:620] *= 2.0 ** (apart - 3)
    dout[:301] *= 2.0 ** -3
    dout[620:] *= 2.0 ** -3
    dout[620:, : H // HK] *= 2.0 ** apart
    q, k, v, dout = _half(q, k, v, dout.clamp(-60000, 60000))
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    _compare(q, k, v, dout, _train(q, k, v, dout, cu), ends)


@pytest.mark.parametrize("N,H,HK,D", SIZES)
def test_rows_of_different_weight(N, H, HK, D):
    """Rows of dO 2^0, 2^-5, .. apart from row to row, the largest first; every seventh row of v 2^8 above the rest."""
    q, k, v, dout = _inputs(N, H, HK, D, N + 3 * D)
    row = torch.arange(N, device=DEV)[:, None, None]
    dout = dout * 2.0 ** (10 - 5 * (row % 4) - 3 * (4 * row // N))
    v = v * torch.where(row % 7 == 3, 2.0 ** 8, 1.0)
    q, k, v, dout = _half(q, k, v, dout)
    cu = torch.tensor([0, N], dtype=torch.int32, device=DEV)
    _compare(q, k, v, dout, _train(q, k, v, dout, cu), [0, N])


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_rows_behind_an_infinity(bad):
    """Keys behind a row of dO that holds an infinity or NaN, and queries before a value that does, keep their precision."""
    q, k, v, dout = _half(*_inputs(400, 4, 2, 64, 9))
    d2, v2 = dout.clone(), v.clone()
    d2[130, :, 3] = bad
    v2[270, :, 5] = bad
    cu = torch.tensor([0, 400], dtype=torch.int32, device=DEV)
    out, dq, dk, dv = _train(q, k, v, d2, cu)
    _compare(q, k, v, dout, (out, torch.cat((dq[:130], dq[131:])), dk, dv), [0, 400], names=("out",))
    for hk in range(2):
        hs = slice(2 * hk, 2 * hk + 2)
        want = exact(q[:, hs], k[:, hk], v[:, hk], dout[:, hs], 0.125)
        for x, (value, bound) in ((dk, want["dk"]), (dv, want["dv"])):
            assert ((x[131:, hk].double() - value[131:]).abs() <= bound[131:]).all()
    out, dq, dk, dv = _train(q, k, v2, dout, cu)
    for hk in range(2):
        hs = slice(2 * hk, 2 * hk + 2)
        value, bound = exact(q[:, hs], k[:, hk], v[:, hk], dout[:, hs], 0.125)["dq"]
        assert ((dq[:270, hs].double() - value[:270]).abs() <= bound[:270]).all()


@pytest.mark.parametrize("N,H,HK,D", [(4096, 1, 1, 64), (2000, 2, 1, 128), (3000, 48, 6, 64)])
def test_values_of_small_weights(N, H, HK, D):
    """Peaked scores: weights far below fp16's smallest normal number add up in dV."""
    q, k, v, dout = _half(*_inputs(N, H, HK, D, 21, std=1.5))
    got = _train(q, k, v, dout, torch.tensor([0, N], dtype=torch.int32, device=DEV))
    if HK > 1:
        G = H // HK
        q, dout, got = q[:, -G:], dout[:, -G:], (got[0][:, -G:], got[1][:, -G:], got[2][:, -1:], got[3][:, -1:])
        k, v = k[:, -1:], v[:, -1:]
    _compare(q, k, v, dout, got, [0, N])


@pytest.mark.parametrize("N,D,H", [(4096, 64, 2), (2500, 128, 3)])
def test_values_of_vanishing_weights(N, D, H):
    """A key whose weights are all below 2^-25 has a gradient of its value all the same."""
    g = torch.Generator().manual_seed(D)
    q = torch.zeros(N, H, D, dtype=FP16, device=DEV)
    k = torch.zeros(N, 1, D, dtype=FP16, device=DEV)
    q[..., 0], k[40::60, :, 0] = 1, -11
    v, dout = (torch.randn(N, h, D, generator=g).to(DEV).half() for h in (1, H))
    dout = 32 * (dout.abs() + 1)
    got = _train(q, k, v, dout, torch.tensor([0, N], dtype=torch.int32, device=DEV), 1.0)
    _compare(q, k, v, dout, got, [0, N], names=("dv",), scale=1.0)


@pytest.mark.parametrize("N,H,HK,D", [(260, 4, 2, 64), (1030, 128, 4, 64)])
def test_wanted_gradients_streams_and_replays(N, H, HK, D):
    """Gradients do not depend on which are wanted, nor on the stream; a captured call follows its inputs."""
    q, k, v, dout = _half(*_inputs(N, H, HK, D, 5))
    cu = torch.tensor([0, N // 3, N], dtype=torch.int32, device=DEV)

    def call(needs=(True, True, True)):
        out, lse, low = sa.causal_attention_forward(q, k, v, cu, keep_low=True)
        return sa.causal_attention_backward(q, k, v, out, lse, dout, cu, needs=needs, out_low=low)

    want = call()
    for mask in range(1, 8):
        needs = [bool(mask >> i & 1) for i in range(3)]
        for need, a, b in zip(needs, call(needs), want):
            assert torch.equal(a, b) if need else a is None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    g = torch.Generator().manual_seed(6)
    for ends, size in (([0, 1, N], 1.0), ([0, N // 2, N // 2], 300.0), ([5, 70, N - 3], 2.0 ** -10)):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        for x in (q, k, v, dout):
            x.copy_(torch.randn(x.shape, generator=g))
        v.mul_(size)
        dout.mul_(size)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        assert all(torch.equal(a, b) for a, b in zip(got, call()))
        for x in got:                                        # (of v and dO of 300, dS k exceeds 65504: infinities, but no NaN)
            assert not torch.isnan(x).any()

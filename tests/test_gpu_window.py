"""causal_attention with a window and first keys that stay visible, against the definition in 64 bits (bounds: window_util.py):
types, head layouts, lengths and windows from one on, packed sequences, views, values that must not reach rows which do not
see them, gradients against differences, other streams, graphs."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib
from tests.causal_util import check
from tests.window_util import exact, sees

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(lead, H, HK, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*lead, h, D, generator=g) * s).to(dtype).to(DEV) for h, s in ((H, std), (HK, std), (HK, 1.0), (H, 1.0))]


def _rounded(dtype, flags=0):
    return dtype != FP32 and not flags


def _compare(q, k, v, dout, out, lse, grads, spans, scale, dtype, flags, window, sinks):
    """spans: (index of the rows, index of the lse) of each sequence."""
    H, HK = q.shape[-2], k.shape[-2]
    G = H // HK
    for rows, lrows in spans:
        for hk in range(HK):
            hs = slice(hk * G, hk * G + G)
            want = exact(q[rows][:, hs], k[rows][:, hk], v[rows][:, hk], dout[rows][:, hs], scale, dtype, _rounded(dtype, flags), window, sinks)
            check(out[rows][:, hs], want["out"], "out")
            check(lse[lrows][..., :][hs].transpose(0, 1), want["lse"], "lse")
            if grads is not None:
                check(grads[0][rows][:, hs], want["dq"], "dq")
                check(grads[1][rows][:, hk:hk + 1], want["dk"], "dk")
                check(grads[2][rows][:, hk:hk + 1], want["dv"], "dv")


def _all(q, k, v, dout, window, sinks, flags=0, cu=None, scale=None):
    out, lse, low = sa.causal_attention_forward(q, k, v, cu, scale, flags=flags, keep_low=True, window=window, sinks=sinks)
    return out, lse, sa.causal_attention_backward(q, k, v, out, lse, dout, cu, scale, flags=flags, out_low=low, window=window, sinks=sinks)


SHAPES = [(1, 2, 1, 1, 64, 1, 0), (2, 3, 2, 1, 64, 2, 1), (1, 31, 3, 3, 32, 5, 0), (1, 33, 4, 2, 128, 32, 1), (2, 64, 2, 2, 64, 33, 4),
          (1, 65, 8, 1, 128, 64, 0), (1, 127, 2, 1, 80, 31, 40), (1, 129, 6, 2, 128, 1, 3), (2, 200, 4, 4, 64, 64, 65), (1, 257, 4, 1, 128, 128, 4),
          (1, 300, 2, 1, 96, 17, 0), (1, 511, 2, 2, 128, 200, 130), (1, 1000, 2, 1, 64, 512, 4), (1, 777, 3, 1, 128, 100, 1), (1, 1300, 8, 2, 128, 300, 2),
          (1, 640, 4, 1, 64, 96, 33), (1, 70, 2, 1, 8, 20, 3), (1, 200, 2, 1, 256, 40, 5), (1, 177, 2, 2, 136, 129, 0), (1, 50, 1, 1, 33, 7, 2),
          (1, 45, 2, 1, 1, 3, 3), (1, 300, 2, 1, 250, 60, 40), (1, 333, 3, 1, 161, 90, 2), (1, 900, 2, 1, 256, 300, 140), (1, 130, 2, 1, 64, 129, 0), (2, 1100, 16, 4, 128, 512, 4), (1, 600, 5, 1, 64, 256, 150)]


@pytest.mark.parametrize("flags", [_lib.FLAG_AUTO, _lib.FLAG_FORCE_GENERIC])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,N,H,HK,D,window,sinks", SHAPES)
def test_batches(B, N, H, HK, D, window, sinks, dtype, flags):
    if dtype == FP32 and flags:
        pytest.skip("the same kernels")
    q, k, v, dout = _inputs((B, N), H, HK, D, dtype, B + N + D)
    out, lse, grads = _all(q, k, v, dout, window, sinks, flags)
    _compare(q, k, v, dout, out, lse, grads, [((b,), (b,)) for b in range(B)], D ** -0.5, dtype, flags, window, sinks)


PACKED = [[0, 5], [0, 1, 2, 3], [0, 0, 64, 64, 65, 200], [3, 40, 40, 168, 297], [0, 300, 301, 900], [0, 1030, 1031, 1600]]


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 0), (20, 3), (64, 0), (150, 70)])
@pytest.mark.parametrize("dtype,H,HK,D", [(BF16, 4, 1, 128), (FP16, 2, 1, 64), (FP32, 3, 3, 64), (BF16, 2, 2, 40), (FP32, 2, 1, 128), (BF16, 1, 1, 256)])
@pytest.mark.parametrize("ends", PACKED)
def test_packed(ends, dtype, H, HK, D, window, sinks):
    T = ends[-1] + 9
    q, k, v, dout = _inputs((T,), H, HK, D, dtype, T + D)
    for x in (q, k, v, dout):                                # rows of no sequence hold anything
        x[:ends[0]] = math.nan
        x[ends[-1]:] = math.inf
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    out, lse, grads = _all(q, k, v, dout, window, sinks, 0, cu)
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, D ** -0.5, dtype, 0, window, sinks)
    for x in (out, *grads):
        assert x[:ends[0]].count_nonzero() == 0 and x[ends[-1]:].count_nonzero() == 0
    assert (lse[:, ends[-1]:] == -math.inf).all() and (lse[:, :ends[0]] == -math.inf).all()


def test_many_short_sequences():
    """More sequences than a wavefront has lanes, some empty."""
    g = torch.Generator().manual_seed(2)
    ends = [0]
    for n in torch.randint(0, 9, (200,), generator=g).tolist():
        ends.append(ends[-1] + n)
    q, k, v, dout = _inputs((ends[-1],), 2, 1, 64, BF16, 7)
    out, lse, grads = _all(q, k, v, dout, 3, 1, 0, torch.tensor(ends, dtype=torch.int32, device=DEV))
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, 64 ** -0.5, BF16, 0, 3, 1)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("flags", [0, _lib.FLAG_FORCE_GENERIC])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 0), (100, 75), (70, 6)])
def test_hidden_rows_may_hold_anything(dtype, flags, D, window, sinks):
    """An infinity or NaN in row j of k, v, q or dout changes nothing that row j is hidden from."""
    N, at = 300, 70
    q, k, v, dout = _inputs((1, N), 2, 1, D, dtype, 5)
    seen = sees(N, window, sinks)
    queries, keys = seen[:, at].to(DEV), seen[at].to(DEV)    # that see key `at`; that query `at` sees

    def same(a, b):
        # sums of at most 2 N terms in another order: 2 (2 N + 16) e of magnitudes that stay below 64, then one rounding each
        return ((a.double() - b.double()).abs() <= torch.finfo(a.dtype).eps * b.double().abs() + 2 * (2 * N + 16) * 2.0 ** -24 * 64).all()

    base = _all(q, k, v, dout, window, sinks, flags)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[:, at, :, 3], v2[:, at, :, 5] = bad, bad
        out, lse, (dq, _, _) = _all(q, k2, v2, dout, window, sinks, flags)
        assert same(out[:, ~queries], base[0][:, ~queries]) and same(lse[..., ~queries], base[1][..., ~queries]) and same(dq[:, ~queries], base[2][0][:, ~queries])
        assert not torch.isfinite(out[:, queries]).all(-1).any()
        q2, d2 = q.clone(), dout.clone()
        q2[:, at, :, 3], d2[:, at, :, 5] = bad, bad
        _, _, (_, dk, dv) = _all(q2, k, v, d2, window, sinks, flags)
        assert same(dk[:, ~keys], base[2][1][:, ~keys]) and same(dv[:, ~keys], base[2][2][:, ~keys])
        assert not torch.isfinite(dv[:, keys].float()).all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_of_any_size(dtype, D):
    """Scores far above a query's own and the first ones it meets; rows of scores that are all very low."""
    N, window, sinks = 400, 130, 2
    q, k, v, dout = _inputs((1, N), 4, 2, D, dtype, 11)
    k[:, 100:140] *= 6.0
    q[:, 200:230] *= 4.0
    k[:, 0] *= 8.0
    out, lse, grads = _all(q, k, v, dout, window, sinks)
    _compare(q, k, v, dout, out, lse, grads, [((0,), (0,))], D ** -0.5, dtype, 0, window, sinks)
    out, lse, grads = _all(q, k, v, dout, window, sinks, scale=-0.3)
    _compare(q, k, v, dout, out, lse, grads, [((0,), (0,))], -0.3, dtype, 0, window, sinks)


def test_a_window_over_everything_is_none():
    q, k, v, dout = _inputs((2, 200), 4, 2, 128, BF16, 3)
    plain = _all(q, k, v, dout, None, 0)
    for window, sinks in ((200, 0), (1 << 40, 7), (500, 3)):
        wide = _all(q, k, v, dout, window, sinks)
        assert all(torch.equal(a, b) for a, b in zip((*plain[:2], *plain[2]), (*wide[:2], *wide[2])))
    # packed sequences shorter than the window, in a call longer than it: other kernels, the same masks
    cu = torch.tensor([0, 150, 200], dtype=torch.int32, device=DEV)
    x = [t[0] for t in (q, k, v, dout)]
    out, lse, grads = _all(*x, 160, 5, 0, cu)
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in ((0, 150), (150, 200))]
    _compare(*x, out, lse, grads, spans, 128 ** -0.5, BF16, 0, 160, 5)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_views_and_wanted_gradients(dtype):
    """q, k and v as views of one projection, rows off the grid, each gradient alone, through autograd."""
    g = torch.Generator().manual_seed(9)
    for width, flags in ((0, 0), (1, 0)):
        fused = torch.randn(2, 300, 4 + 2 * 2, 64 + width, generator=g).to(dtype).to(DEV)[..., width:]
        views = [fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:]]
        dout = torch.randn(2, 4, 300, 64, generator=g).to(dtype).to(DEV).transpose(1, 2)
        whole = [t.contiguous() for t in views]
        out, lse, grads = _all(*whole, dout.contiguous(), 90, 3, _lib.FLAG_FORCE_GENERIC if width else 0)
        for needs in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)):
            leaves = [t.detach().requires_grad_(bool(n)) for t, n in zip(views, needs)]
            o = sa.causal_attention(*leaves, window=90, sinks=3)
            got = torch.autograd.grad(o, [t for t in leaves if t.requires_grad], dout)
            assert torch.equal(o, out)
            assert all(torch.equal(a, b) for a, b in zip(got, [x for x, n in zip(grads, needs) if n]))


def test_gradients_against_differences():
    """fp32: the derivative along a direction, from two calls at +- h (h^2 of the third derivative and rounding / h are left)."""
    q, k, v, dout = _inputs((1, 130), 2, 1, 64, FP32, 21)
    dirs = _inputs((1, 130), 2, 1, 64, FP32, 22)[:3]
    _, _, grads = _all(q, k, v, dout, 30, 2)
    h = 2.0 ** -6
    for i, x in enumerate((q, k, v)):
        def at(s):
            a = [q, k, v]
            a[i] = x + s * h * dirs[i]
            return (sa.causal_attention(*a, window=30, sinks=2).double() * dout.double()).sum()
        slope = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * h)
        want = (grads[i].double() * dirs[i].double()).sum()
        # h^4 / 30 of the fifth derivative (of a few thousand terms of size one), and fp32 outputs' rounding over h
        assert (slope - want).abs() <= 2e-3 * (1 + want.abs())


def test_other_streams_and_graphs():
    q, k, v, dout = _inputs((1, 500), 4, 1, 128, BF16, 31)
    want = _all(q, k, v, dout, 100, 4)
    flat = lambda r: (*r[:2], *r[2])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all(q, k, v, dout, 100, 4)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(want)))
    static = [torch.empty_like(t) for t in (q, k, v, dout)]
    graph = torch.cuda.CUDAGraph()
    for t, x in zip(static, (q, k, v, dout)):
        t.copy_(x)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = _all(*static, 100, 4)
    for seed in (1, 2, 3):
        x = _inputs((1, 500), 4, 1, 128, BF16, seed)
        for t, y in zip(static, x):
            t.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(flat(got), flat(_all(*x, 100, 4))))


def test_results_are_deterministic():
    q, k, v, dout = _inputs((1, 3000), 8, 2, 128, BF16, 41)
    first = _all(q, k, v, dout, 256, 4)
    second = _all(q, k, v, dout, 256, 4)
    assert all(torch.equal(a, b) for a, b in zip((*first[:2], *first[2]), (*second[:2], *second[2])))


def test_tensors_of_more_than_2_to_31_elements():
    """The last rows of a long sequence against those rows by themselves: without first keys they see nothing else."""
    N, H, HK, D, window, rows = 270_000, 64, 8, 128, 100, 300
    g = torch.Generator(device=DEV).manual_seed(5)
    q, k, v, dout = (torch.empty(1, N, h, D, dtype=BF16, device=DEV).normal_(generator=g) for h in (H, HK, HK, H))
    out, lse, grads = _all(q, k, v, dout, window, 0)
    near, at = slice(N - rows - window + 1, N), slice(window - 1, None)
    for hk in (0, HK - 1):
        hs = slice(8 * hk, 8 * hk + 8)
        want = exact(q[0, near, hs], k[0, near, hk], v[0, near, hk], dout[0, near, hs], D ** -0.5, BF16, True, window, 0)
        check(out[0, near, hs][at], [x[at] for x in want["out"]], "out")
        check(lse[0, hs, near].transpose(0, 1)[at], [x[at] for x in want["lse"]], "lse")
        check(grads[0][0, near, hs][at], [x[at] for x in want["dq"]], "dq")
        check(grads[1][0, near, hk:hk + 1][at], [x[at] for x in want["dk"]], "dk")
        check(grads[2][0, near, hk:hk + 1][at], [x[at] for x in want["dv"]], "dv")

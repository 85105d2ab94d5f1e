"""Windowed attention where a wavefront has two blocks of 32 queries (calls of 512 workgroups and more: sizes that serving and training run),
against the definition in 64 bits (bounds: window_util.py): head layouts, first keys, packed rows, hidden rows that hold anything, large scores."""
import math

import pytest
import torch

from tests.causal_util import check
from tests.test_gpu_window import BF16, DEV, FP16, _all, _compare, _inputs
from tests.window_util import exact, sees

pytestmark = pytest.mark.gpu

# workgroups of 512 and more: batch * heads / (2 or 4 that share one) * blocks of 64, 128 or 256 queries
SHAPES = [(70, 513, 4, 1, 128, 100, 4), (110, 700, 2, 1, 64, 130, 70), (40, 1100, 8, 2, 128, 512, 4), (180, 600, 1, 1, 80, 300, 0), (300, 200, 2, 2, 64, 40, 3),
          (30, 1500, 4, 4, 32, 64, 33), (8, 5000, 4, 1, 128, 1000, 200), (520, 65, 4, 1, 64, 33, 1), (600, 31, 4, 1, 128, 7, 2), (170, 400, 3, 1, 128, 1, 0),
          (60, 640, 4, 1, 64, 512, 129), (9, 4000, 4, 1, 64, 700, 4), (90, 450, 6, 3, 96, 449, 1), (260, 129, 8, 2, 8, 128, 0)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,N,H,HK,D,window,sinks", SHAPES)
def test_batches(B, N, H, HK, D, window, sinks, dtype):
    q, k, v, dout = _inputs((B, N), H, HK, D, dtype, B + N + D)
    out, lse, grads = _all(q, k, v, dout, window, sinks)
    _compare(q, k, v, dout, out, lse, grads, [((b,), (b,)) for b in (0, B // 2, B - 1)], D ** -0.5, dtype, 0, window, sinks)
    again = _all(q, k, v, dout, window, sinks)
    assert all(torch.equal(a, b) for a, b in zip((out, lse, *grads), (*again[:2], *again[2])))


@pytest.mark.parametrize("window,sinks", [(20, 3), (64, 0), (150, 70), (300, 4)])
@pytest.mark.parametrize("dtype,H,HK,D", [(BF16, 4, 1, 128), (FP16, 4, 1, 128), (FP16, 4, 2, 64), (BF16, 2, 2, 40)])
def test_packed(dtype, H, HK, D, window, sinks):
    g = torch.Generator().manual_seed(window)
    lengths = torch.randint(0, 200, (400,), generator=g).tolist()
    lengths[3], lengths[100], lengths[399] = 2000, 1, 777
    ends = [5]
    for n in lengths:
        ends.append(ends[-1] + n)
    q, k, v, dout = _inputs((ends[-1] + 9,), H, HK, D, dtype, ends[-1] + D)
    for x in (q, k, v, dout):                                # rows of no sequence hold anything
        x[:ends[0]] = math.nan
        x[ends[-1]:] = math.inf
    out, lse, grads = _all(q, k, v, dout, window, sinks, 0, torch.tensor(ends, dtype=torch.int32, device=DEV))
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans[:8] + spans[90:110] + spans[-6:], D ** -0.5, dtype, 0, window, sinks)
    for x in (out, *grads):
        assert x[:ends[0]].count_nonzero() == 0 and x[ends[-1]:].count_nonzero() == 0
    assert (lse[:, ends[-1]:] == -math.inf).all() and (lse[:, :ends[0]] == -math.inf).all()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,sinks", [(40, 0), (300, 75), (200, 6)])
def test_hidden_rows_may_hold_anything(dtype, D, window, sinks):
    """An infinity or NaN in row j of k, v, q or dout changes nothing that row j is hidden from."""
    B, N, at = 60, 600, 70
    q, k, v, dout = _inputs((B, N), 4, 1, D, dtype, 5)
    seen = sees(N, window, sinks)
    queries, keys = seen[:, at].to(DEV), seen[at].to(DEV)    # that see key `at`; that query `at` sees

    some = (0, 31, B - 1)
    want = [exact(q[b], k[b, :, 0], v[b, :, 0], dout[b], D ** -0.5, dtype, True, window, sinks) for b in some]
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[:, at, :, 3], v2[:, at, :, 5] = bad, bad
        out, lse, (dq, _, _) = _all(q, k2, v2, dout, window, sinks)
        q2, d2 = q.clone(), dout.clone()
        q2[:, at, :, 3], d2[:, at, :, 5] = bad, bad
        _, _, (_, dk, dv) = _all(q2, k, v, d2, window, sinks)
        for b, w in zip(some, want):
            for got, name, rows in ((out[b], "out", ~queries), (lse[b].T, "lse", ~queries), (dq[b], "dq", ~queries), (dk[b], "dk", ~keys), (dv[b], "dv", ~keys)):
                check(got[rows], [x[rows] for x in w[name]], name)
        assert not torch.isfinite(out[:, queries]).all(-1).any() and not torch.isfinite(dv[:, keys].float()).all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_scores_of_any_size(dtype, D):
    """Scores far above a query's own and the first ones it meets; rows of scores that are all very low."""
    B, N, window, sinks = 80, 420, 130, 2
    q, k, v, dout = _inputs((B, N), 4, 1, D, dtype, 11)
    k[:, 100:140] *= 6.0
    q[:, 200:230] *= 4.0
    k[:, 0] *= 8.0
    for scale in (None, -0.3):
        out, lse, grads = _all(q, k, v, dout, window, sinks, scale=scale)
        _compare(q, k, v, dout, out, lse, grads, [((b,), (b,)) for b in (0, 41, B - 1)], scale or D ** -0.5, dtype, 0, window, sinks)


def test_graphs():
    q, k, v, dout = _inputs((70, 520), 4, 1, 64, FP16, 31)
    static = [t.clone() for t in (q, k, v, dout)]
    _all(*static, 100, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _all(*static, 100, 4)
    for seed in (1, 2, 3):
        x = _inputs((70, 520), 4, 1, 64, FP16, seed)
        for t, y in zip(static, x):
            t.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = _all(*x, 100, 4)
        assert all(torch.equal(a, b) for a, b in zip((*got[:2], *got[2]), (*want[:2], *want[2])))

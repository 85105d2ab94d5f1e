"""causal_attention without a window at head_dims above 128 and sequences longer than a workgroup's 128 rows (kernels with fp32 products),
against the definition in 64 bits (bounds: window_util.py, with a window over everything)."""
import math

import pytest
import torch

from simplical_attn_amd import _lib
from tests.causal_util import check
from tests.test_gpu_window import BF16, DEV, FP16, FP32, _all, _compare, _inputs
from tests.window_util import exact, sees

pytestmark = pytest.mark.gpu

SHAPES = [(1, 177, 1, 1, 136), (1, 177, 2, 2, 136), (1, 300, 4, 2, 129), (2, 257, 3, 1, 161), (1, 511, 2, 1, 192), (1, 900, 2, 2, 200), (1, 385, 6, 2, 250), (1, 640, 4, 1, 256), (1, 129, 2, 1, 255), (1, 1100, 2, 1, 144)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,N,H,HK,D", SHAPES)
def test_batches(B, N, H, HK, D, dtype):
    q, k, v, dout = _inputs((B, N), H, HK, D, dtype, B + N + D)
    out, lse, grads = _all(q, k, v, dout, None, 0)
    _compare(q, k, v, dout, out, lse, grads, [((b,), (b,)) for b in range(B)], D ** -0.5, dtype, _lib.FLAG_FORCE_GENERIC, N, 0)


@pytest.mark.parametrize("dtype,D", [(BF16, 136), (FP32, 250), (FP32, 136), (FP16, 256)])
@pytest.mark.parametrize("ends", [[0, 300, 301, 900], [3, 40, 40, 168, 497], [0, 0, 64, 264, 265, 600]])
def test_packed(ends, dtype, D):
    q, k, v, dout = _inputs((ends[-1] + 9,), 4, 2, D, dtype, ends[-1] + D)
    for x in (q, k, v, dout):
        x[:ends[0]], x[ends[-1]:] = math.nan, math.inf
    out, lse, grads = _all(q, k, v, dout, None, 0, 0, torch.tensor(ends, dtype=torch.int32, device=DEV))
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, D ** -0.5, dtype, _lib.FLAG_FORCE_GENERIC, ends[-1], 0)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("D", [136, 256])
@pytest.mark.parametrize("at", [70, 130, 255])
def test_hidden_rows_may_hold_anything(dtype, D, at):
    N = 400
    q, k, v, dout = _inputs((1, N), 2, 1, D, dtype, 5)
    seen = sees(N, N, 0)
    queries, keys = seen[:, at].to(DEV), seen[at].to(DEV)    # that see key `at`; that query `at` sees
    want = exact(q[0], k[0, :, 0], v[0, :, 0], dout[0], D ** -0.5, dtype, False, N, 0)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2, q2, d2 = k.clone(), v.clone(), q.clone(), dout.clone()
        k2[:, at, :, 3], v2[:, at, :, 5] = bad, bad
        q2[:, at, :, 3], d2[:, at, :, 5] = bad, bad
        out, lse, (dq, _, _) = _all(q, k2, v2, dout, None, 0)
        _, _, (_, dk, dv) = _all(q2, k, v, d2, None, 0)
        for got, name, rows in ((out[0], "out", ~queries), (lse[0].T, "lse", ~queries), (dq[0], "dq", ~queries), (dk[0], "dk", ~keys), (dv[0], "dv", ~keys)):
            check(got[rows], [x[rows] for x in want[name]], name)

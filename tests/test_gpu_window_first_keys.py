"""Windowed attention of many short packed sequences with more first keys than most of them have rows, against the definition in 64 bits:
their gradients' sums lie by rows."""
import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib
from tests.test_gpu_window import BF16, DEV, FP16, FP32, _all, _compare, _inputs

pytestmark = pytest.mark.gpu


def _ends(lengths):
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


def _check_packed(ends, H, HK, D, dtype, window, sinks, flags=0, behind=7):
    q, k, v, dout = _inputs((ends[-1] + behind,), H, HK, D, dtype, ends[-1] + D)
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    results = [_all(q, k, v, dout, window, sinks, flags, cu) for _ in range(2)]
    out, lse, grads = results[0]
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, D ** -0.5, dtype, flags, window, sinks)
    for x, y in zip((out, *grads), (results[1][0], *results[1][2])):
        assert x[ends[-1]:].count_nonzero() == 0 and torch.equal(x, y)


@pytest.mark.parametrize("window,sinks", [(1, 40), (20, 128), (20, 300), (150, 129), (33, 65535)])
@pytest.mark.parametrize("dtype,H,HK,D,flags", [(BF16, 4, 2, 128, 0), (FP16, 2, 1, 64, 0), (FP32, 2, 2, 64, 0), (FP32, 2, 1, 128, 0), (BF16, 3, 1, 256, 0), (FP16, 2, 2, 40, 0),
                                                (BF16, 4, 1, 72, _lib.FLAG_FORCE_GENERIC)])
def test_short_and_long_sequences(dtype, H, HK, D, flags, window, sinks):
    g = torch.Generator().manual_seed(sinks)
    lengths = torch.randint(0, 60, (50,), generator=g).tolist()
    lengths[7], lengths[20], lengths[33], lengths[49] = 700, 129, 128, 300
    _check_packed(_ends(lengths), H, HK, D, dtype, window, sinks, flags)


@pytest.mark.parametrize("lengths", [[1] * 300, [0, 2] * 100, [257, 1, 1, 0, 1], [600] + [1] * 70])
def test_the_shortest_sequences(lengths):
    for dtype, sinks in ((BF16, 200), (FP32, 256)):
        _check_packed(_ends(lengths), 2, 1, 64, dtype, 2, sinks)


def test_gradients_that_are_wanted_alone():
    ends = _ends([30, 0, 200, 5, 31, 64] * 8)
    q, k, v, dout = _inputs((ends[-1],), 4, 2, 64, BF16, 3)
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    for flags in (0, _lib.FLAG_FORCE_GENERIC):
        out, lse, low = sa.causal_attention_forward(q, k, v, cu, flags=flags, keep_low=True, window=9, sinks=150)
        run = lambda needs: sa.causal_attention_backward(q, k, v, out, lse, dout, cu, needs=needs, flags=flags, out_low=low, window=9, sinks=150)  # noqa: E731
        whole = run((True, True, True))
        for needs in ((True, False, False), (False, True, False), (False, False, True)):
            for got, want, wanted in zip(run(needs), whole, needs):
                assert torch.equal(got, want) if wanted else got is None


def test_bounds_out_of_order():
    """No defined gradients, but no access outside of the tensors either."""
    q, k, v, dout = _inputs((400,), 2, 1, 64, BF16, 3)
    for ends in ([0, 100, 200, 50] * 30, [-7, 500, 300, 90] * 30, [300, 200, 100, 0] * 30, [0, 399, 10, 380] * 30):
        for dtype in (BF16, FP32):
            x = [t.to(dtype) for t in (q, k, v, dout)]
            _all(*x, 20, 150, 0, torch.tensor(ends, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()

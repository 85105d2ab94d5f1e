"""causal_attention against the definition in 64 bits (bounds: causal_util.py): types, head layouts, lengths from one row on,
packed sequences with empty ones and rows behind the last, views, values that must not reach rows which do not see them,
gradients against differences, other streams, graphs."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib
from tests.causal_util import check, exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(lead, H, HK, D, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*lead, h, D, generator=g) * s).to(dtype).to(DEV) for h, s in ((H, std), (HK, std), (HK, 1.0), (H, 1.0))]


def _rounded(dtype, flags=0):
    return dtype != FP32 and not flags


def _compare(q, k, v, dout, out, lse, grads, spans, scale, dtype, flags):
    """spans: (index of the rows, index of the lse) of each sequence."""
    H, HK = q.shape[-2], k.shape[-2]
    G = H // HK
    for rows, lrows in spans:
        for hk in range(HK):
            hs = slice(hk * G, hk * G + G)
            want = exact(q[rows][:, hs], k[rows][:, hk], v[rows][:, hk], dout[rows][:, hs], scale, dtype, _rounded(dtype, flags))
            check(out[rows][:, hs], want["out"], "out")
            check(lse[lrows][..., :][hs].transpose(0, 1), want["lse"], "lse")
            if grads is not None:
                check(grads[0][rows][:, hs], want["dq"], "dq")
                check(grads[1][rows][:, hk:hk + 1], want["dk"], "dk")
                check(grads[2][rows][:, hk:hk + 1], want["dv"], "dv")


def _all(q, k, v, dout, flags, cu=None, scale=None):
    out, lse = sa.causal_attention_forward(q, k, v, cu, scale, flags=flags)
    return out, lse, sa.causal_attention_backward(q, k, v, out, lse, dout, cu, scale, flags=flags)


SHAPES = [(1, 1, 1, 1, 64), (2, 2, 2, 1, 64), (1, 31, 3, 3, 32), (1, 33, 4, 2, 128), (2, 64, 2, 2, 64), (1, 65, 8, 1, 128),
          (1, 127, 2, 1, 80), (1, 129, 6, 2, 128), (2, 200, 4, 4, 64), (1, 257, 4, 1, 128), (1, 300, 2, 1, 96), (1, 511, 2, 2, 128),
          (1, 1000, 2, 1, 64), (1, 777, 3, 1, 128), (1, 70, 2, 1, 8), (1, 40, 2, 1, 256), (1, 77, 2, 2, 136), (1, 50, 1, 1, 33), (1, 45, 2, 1, 1)]


@pytest.mark.parametrize("flags", [_lib.FLAG_AUTO, _lib.FLAG_FORCE_GENERIC])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,N,H,HK,D", SHAPES)
def test_batches(B, N, H, HK, D, dtype, flags):
    if dtype == FP32 and flags:
        pytest.skip("the same kernels")
    q, k, v, dout = _inputs((B, N), H, HK, D, dtype, B + N + D)
    out, lse, grads = _all(q, k, v, dout, flags)
    _compare(q, k, v, dout, out, lse, grads, [((b,), (b,)) for b in range(B)], D ** -0.5, dtype, flags)


PACKED = [[0, 5], [0, 1, 2, 3], [0, 0, 64, 64, 65, 200], [3, 40, 40, 168, 297], [0, 300, 301, 900]]


@pytest.mark.parametrize("dtype,H,HK,D", [(BF16, 4, 2, 128), (FP16, 2, 1, 64), (FP32, 3, 3, 64), (BF16, 2, 2, 40), (FP32, 2, 1, 128), (BF16, 1, 1, 256)])
@pytest.mark.parametrize("ends", PACKED)
def test_packed(ends, dtype, H, HK, D):
    T = ends[-1] + 9
    q, k, v, dout = _inputs((T,), H, HK, D, dtype, T + D)
    for x in (q, k, v, dout):                                # rows of no sequence hold anything
        x[:ends[0]] = math.nan
        x[ends[-1]:] = math.inf
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    out, lse, grads = _all(q, k, v, dout, 0, cu)
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, D ** -0.5, dtype, 0)
    for x in (out, *grads):
        assert x[:ends[0]].count_nonzero() == 0 and x[ends[-1]:].count_nonzero() == 0
    assert (lse[:, ends[-1]:] == -math.inf).all() and (lse[:, :ends[0]] == -math.inf).all()


def test_many_short_sequences():
    """More sequences than a wavefront has lanes, some empty."""
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 9, (200,), generator=g).tolist()
    ends = [0]
    for n in lens:
        ends.append(ends[-1] + n)
    q, k, v, dout = _inputs((ends[-1],), 2, 1, 64, BF16, 7)
    out, lse, grads = _all(q, k, v, dout, 0, torch.tensor(ends, dtype=torch.int32, device=DEV))
    spans = [((slice(a, b),), (slice(None), slice(a, b))) for a, b in zip(ends, ends[1:]) if b > a]
    _compare(q, k, v, dout, out, lse, grads, spans, 64 ** -0.5, BF16, 0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("flags", [0, _lib.FLAG_FORCE_GENERIC])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_rows_may_hold_anything(dtype, flags, D):
    """An infinity or NaN in row j of k, v, q or dout changes nothing that row j is hidden from."""
    N, at = 150, 70
    q, k, v, dout = _inputs((1, N), 2, 1, D, dtype, 5)

    def same(a, b):
        # sums of at most 2 N terms in another order: 2 (2 N + 16) e of magnitudes that stay below 64, then one rounding each
        return ((a.double() - b.double()).abs() <= torch.finfo(a.dtype).eps * b.double().abs() + 2 * (2 * N + 16) * 2.0 ** -24 * 64).all()

    base = _all(q, k, v, dout, flags)
    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = k.clone(), v.clone()
        k2[:, at, :, 3], v2[:, at, :, 5] = bad, bad
        out, lse, (dq, _, _) = _all(q, k2, v2, dout, flags)
        assert same(out[:, :at], base[0][:, :at]) and same(lse[..., :at], base[1][..., :at]) and same(dq[:, :at], base[2][0][:, :at])
        assert not torch.isfinite(out[:, at:]).all(-1).any()
        q2, d2 = q.clone(), dout.clone()
        q2[:, at, :, 3], d2[:, at, :, 5] = bad, bad
        _, _, (_, dk, dv) = _all(q2, k, v, d2, flags)
        assert same(dk[:, at + 1:], base[2][1][:, at + 1:]) and same(dv[:, at + 1:], base[2][2][:, at + 1:])
        assert not torch.isfinite(dv[:, :at + 1].float()).all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_views_broadcasts_and_odd_rows(dtype):
    g = torch.Generator().manual_seed(11)
    fused = torch.randn(2, 90, 8, 64, generator=g).to(dtype).to(DEV)
    q, k, v = fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:8]
    dout = torch.randn(2, 4, 90, 64, generator=g).to(dtype).to(DEV).transpose(1, 2)
    want = _all(q.contiguous(), k.contiguous(), v.contiguous(), dout.contiguous(), 0)
    got = _all(q, k, v, dout, 0)
    for a, b in zip((*got[:2], *got[2]), (*want[:2], *want[2])):
        assert torch.equal(a, b)
    # a head shared by expansion, a gradient expanded over rows, rows off the 16-byte grid
    wide = torch.randn(1, 70, 2, 70, generator=g).to(dtype).to(DEV)
    q, k = wide[..., 3:67], wide[:, :, :1, 5:69].expand(1, 70, 2, 64)
    dout = torch.ones(1, 1, 1, 1, dtype=dtype, device=DEV).expand(1, 70, 2, 64)
    got = _all(q, k, k, dout, 0)
    # (rows off the grid run on the kernels with fp32 products)
    _compare(q, k, k, dout, got[0], got[1], got[2], [((0,), (0,))], 0.125, dtype, 0)


@pytest.mark.parametrize("scale", [0.0, -0.125, 0.5, 2.0])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_scales(scale, dtype):
    q, k, v, dout = _inputs((1, 140), 2, 2, 64, dtype, 3)
    out, lse, grads = _all(q, k, v, dout, 0, scale=scale)
    _compare(q, k, v, dout, out, lse, grads, [((0,), (0,))], scale, dtype, 0)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_large_scores(dtype):
    """Scores of several hundred: the running maximum moves, weights underflow."""
    q, k, v, dout = _inputs((1, 300), 2, 1, 128, dtype, 13, std=6.0)
    out, lse, grads = _all(q, k, v, dout, 0)
    _compare(q, k, v, dout, out, lse, grads, [((0,), (0,))], 128 ** -0.5, dtype, 0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,N,H,HK,D", [(1, 300, 128, 16, 128), (8, 513, 16, 4, 64), (4, 1100, 16, 16, 128), (3, 700, 32, 8, 80), (2, 1500, 24, 24, 64)])
def test_many_rows(B, N, H, HK, D, dtype):
    """Sizes at which a wavefront owns 64 queries; some heads are compared."""
    q, k, v, dout = _inputs((B, N), H, HK, D, dtype, N + D)
    out, lse, grads = _all(q, k, v, dout, 0)
    G = H // HK
    for b, hk in ((0, 0), (B - 1, HK - 1), (B // 2, HK // 2)):
        hs, ks = slice(hk * G, hk * G + G), slice(hk, hk + 1)
        part = lambda x, heads: x[b:b + 1][:, :, heads]
        _compare(part(q, hs), part(k, ks), part(v, ks), part(dout, hs), part(out, hs), lse[b:b + 1, hs],
                 [part(x, h) for x, h in zip(grads, (hs, ks, ks))], [((0,), (0,))], D ** -0.5, dtype, 0)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,HK,D", [(2, 1, 64), (2, 2, 128), (96, 8, 64), (96, 8, 128)])
def test_later_keys_far_above_the_first(H, HK, D, dtype):
    """Scores that exceed the ones of a row's first 32 keys by e^60 and more: the workgroup sweeps its keys a second time."""
    N = 600
    q, k, v, dout = _inputs((1, N), H, HK, D, dtype, H + D, std=4.0)
    k[:, :32] *= 0.01
    out, lse, grads = _all(q, k, v, dout, 0)
    G = H // HK
    for hk in (0, HK - 1):
        hs, ks = slice(hk * G, hk * G + G), slice(hk, hk + 1)
        _compare(q[:, :, hs], k[:, :, ks], v[:, :, ks], dout[:, :, hs], out[:, :, hs], lse[:, hs], [grads[0][:, :, hs], grads[1][:, :, ks], grads[2][:, :, ks]],
                 [((0,), (0,))], D ** -0.5, dtype, 0)


# blocks of 256 queries: two or more per CU, so that a wavefront owns 64 of them
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,N,H,HK,D", [(1, 300, 256, 16, 128), (16, 513, 12, 4, 64), (8, 1100, 16, 16, 128), (6, 700, 32, 8, 80), (4, 1500, 24, 24, 64), (1, 1023, 144, 8, 64)])
def test_two_blocks_per_wavefront(B, N, H, HK, D, dtype):
    test_many_rows(B, N, H, HK, D, dtype)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("H,HK,D", [(192, 8, 64), (192, 8, 128)])
def test_two_blocks_and_later_keys_far_above_the_first(H, HK, D, dtype):
    test_later_keys_far_above_the_first(H, HK, D, dtype)


# fp32: more blocks of 32 keys than CUs, which make dK and dV together up to head_dim 64
@pytest.mark.parametrize("B,N,H,HK,D", [(4, 600, 8, 4, 64), (2, 700, 16, 8, 32), (3, 450, 8, 4, 50), (2, 600, 8, 4, 128)])
def test_many_rows_of_fp32(B, N, H, HK, D):
    test_many_rows(B, N, H, HK, D, FP32)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_two_blocks_and_hidden_rows(D, dtype):
    """Packed, with rows of no sequence that hold NaN and infinities, and NaN in the last keys and values of each sequence."""
    ends, rows, H, HK = [40, 340, 341, 341, 1100], 1200, 128, 4
    q, k, v, dout = _inputs((rows,), H, HK, D, dtype, 67 + D)
    clean = [t.clone() for t in (q, k, v, dout)]
    for t in (q, k, v, dout):
        t[:40] = math.nan
        t[1100:] = math.inf
    for t in (k, v):
        t[339] = math.nan
        t[1099] = math.inf
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)

    def same(a, b):
        # as in test_hidden_rows_may_hold_anything, with sequences of up to 759 rows
        return ((a.double() - b.double()).abs() <= torch.finfo(a.dtype).eps * b.double().abs() + 2 * (2 * 759 + 16) * 2.0 ** -24 * 64).all()

    out, lse = sa.causal_attention_forward(q, k, v, cu)
    want, want_lse = sa.causal_attention_forward(*clean[:3], cu)
    for lo, hi in ((40, 339), (340, 341), (341, 1099)):
        assert same(out[lo:hi], want[lo:hi]) and same(lse[:, lo:hi], want_lse[:, lo:hi])
    for x in (out[:40], out[1100:]):
        assert x.count_nonzero() == 0
    # gradients of the queries before those keys
    grads = sa.causal_attention_backward(q, k, v, want, want_lse, clean[3], cu)
    clear = sa.causal_attention_backward(*clean[:3], want, want_lse, clean[3], cu)
    for lo, hi in ((40, 339), (340, 341), (341, 1099)):
        assert same(grads[0][lo:hi], clear[0][lo:hi])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_gradients_of_autograd(dtype):
    """The training path, which also keeps what rounding the output left; expanded keys get the sum of their gradients."""
    q, k, v, dout = _inputs((2, 150), 4, 2, 64, dtype, 43)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = sa.causal_attention(*leaves)
    grads = torch.autograd.grad(out, leaves, dout)
    _, lse = sa.causal_attention_forward(q.detach(), k.detach(), v.detach())
    _compare(q.detach(), k.detach(), v.detach(), dout, out.detach(), lse, grads, [((b,), (b,)) for b in range(2)], 0.125, dtype, 0)
    one = k.detach()[:, :, :1].clone().requires_grad_(True)
    (shared,) = torch.autograd.grad(sa.causal_attention(q.detach(), one.expand(2, 150, 4, 64), v.detach()[:, :, :1].expand(2, 150, 4, 64)), one, dout)
    (grouped,) = torch.autograd.grad(sa.causal_attention(q.detach(), one, v.detach()[:, :, :1].contiguous()), one, dout)
    # the four heads' gradients, each rounded to the type and added in it, against the one sum: 8 half steps of their magnitudes
    size = grouped.double().abs().amax()
    assert (shared.double() - grouped.double()).abs().max() <= 8 * torch.finfo(dtype).eps / 2 * 4 * size + 1e-4


def test_small_fp16_gradients():
    """Gradients far below fp16's smallest normal number times the softmax weights keep their precision."""
    q, k, v, dout = _inputs((1, 700), 2, 1, 64, FP16, 47)
    out, lse, want = _all(q, k, v, dout, 0)
    small = (dout.double() * 2.0 ** -9).half()                  # exact: a power of two, above the subnormal numbers for nearly all
    got = sa.causal_attention_backward(q, k, v, out, lse, small)
    for a, b in zip(got[:2], want[:2]):
        # the same up to the rounding of results that are subnormal now (2^-25 each) and of inputs that are
        assert ((a.double() * 2.0 ** 9 - b.double()).abs() <= 2.0 ** -10 * b.double().abs() + 2.0 ** -14 * b.double().abs().max() + 2.0 ** -15).all()


def test_calls_at_once():
    """Two streams, and two captured graphs replayed in turn, each with its own data."""
    sets = [_inputs((1, 260), 4, 2, 64, BF16, 50 + i) for i in range(2)]
    want = [_all(*x, 0) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        got = []
        for st, x in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_all(*x, 0))
    torch.cuda.synchronize()
    graphs, captured = [], []
    for x in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            captured.append(_all(*x, 0))
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for results in (got, captured):
        for r, w in zip(results, want):
            for a, b in zip((*r[:2], *r[2]), (*w[:2], *w[2])):
                assert torch.equal(a, b)


def test_only_wanted_gradients_and_determinism():
    q, k, v, dout = _inputs((1, 400), 4, 2, 64, BF16, 17)
    out, lse, grads = _all(q, k, v, dout, 0)
    for mask in range(8):
        needs = [bool(mask >> i & 1) for i in range(3)]
        got = sa.causal_attention_backward(q, k, v, out, lse, dout, needs=needs)
        for need, a, b in zip(needs, got, grads):
            assert torch.equal(a, b) if need else a is None
    leaf = v.clone().requires_grad_(True)
    (dv,) = torch.autograd.grad(sa.causal_attention(q, k, leaf), leaf, dout)
    assert torch.equal(dv, grads[2])


def test_gradients_against_differences():
    q, k, v, dout = _inputs((1, 40), 4, 2, 64, FP32, 19)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(sa.causal_attention(*leaves), leaves, dout)
    f = lambda *x: (sa.causal_attention(*x).double() * dout.double()).sum().item()
    g = torch.Generator().manual_seed(20)
    for i, grad in enumerate(grads):
        step = torch.randn(leaves[i].shape, generator=g).to(DEV)
        h = 2.0 ** -6
        moved = [[(t + s * h * step).detach() if j == i else t.detach() for j, t in enumerate(leaves)] for s in (1, -1)]
        slope = (f(*moved[0]) - f(*moved[1])) / (2 * h)
        # third derivatives are of the order of the gradient itself: h^2; rounding of 10^4 outputs: 10^2 * 2^-24 / h
        size = (grad.double().abs() * step.double().abs()).sum().item()
        assert abs(slope - (grad.double() * step.double()).sum().item()) <= 4 * h * h * size + 1e-3


def test_offsets_beyond_32_bits():
    """Rows 2^31 and more elements into a packed tensor."""
    D, H = 128, 1
    T = (1 << 31) // (8 * D) + 300
    big = torch.zeros(T, 8, D, dtype=BF16, device=DEV)                    # head 0 of 8: rows 1024 elements apart
    q, k, v, dout = _inputs((260,), 1, 1, D, BF16, 23)
    for i, x in enumerate((q, k, v, dout)):
        big[T - 260:, i] = x[:, 0]
    views = [big[:, i:i + 1] for i in range(4)]
    cu = torch.tensor([T - 260, T], dtype=torch.int32, device=DEV)
    out, lse, grads = _all(*views, 0, cu)
    # (a call on the 260 rows alone may take other kernels, so the definition is what the bits are compared with)
    for a in (out, *grads):
        assert a[:T - 260].count_nonzero() == 0
    _compare(q, k, v, dout, out[T - 260:], lse[:, T - 260:].contiguous(), [x[T - 260:] for x in grads],
             [((slice(None),), (slice(None),))], D ** -0.5, BF16, 0)


def test_other_stream_and_replayed_graph():
    q, k, v, dout = _inputs((100,), 4, 2, 128, BF16, 29)
    cu = torch.tensor([0, 30, 100], dtype=torch.int32, device=DEV)
    want = _all(q, k, v, dout, 0, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _all(q, k, v, dout, 0, cu)
    side.synchronize()
    for a, b in zip((*got[:2], *got[2]), (*want[:2], *want[2])):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = _all(q, k, v, dout, 0, cu)
    g = torch.Generator().manual_seed(31)
    for ends in ([0, 1, 100], [0, 64, 64], [50, 80, 99]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        for x in (q, k, v, dout):
            x.copy_(torch.randn(x.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*captured[:2], *captured[2])]
        eager = _all(q, k, v, dout, 0, cu)
        for a, b in zip(got, (*eager[:2], *eager[2])):
            assert torch.equal(a, b)


def test_second_derivatives_are_refused():
    q, k, v, dout = _inputs((1, 40), 2, 1, 64, BF16, 61)
    q.requires_grad_(True)
    out = sa.causal_attention(q, k, v)
    with pytest.raises(RuntimeError, match="first derivatives"):
        torch.autograd.grad(out, q, dout, create_graph=True)


def test_no_query_heads():
    q = torch.zeros(1, 5, 0, 64, dtype=BF16, device=DEV)
    k = torch.ones(1, 5, 2, 64, dtype=BF16, device=DEV, requires_grad=True)
    out = sa.causal_attention(q, k, k)
    assert out.shape == q.shape and torch.autograd.grad(out, k, q)[0].count_nonzero() == 0


def test_empty():
    q = torch.zeros(2, 0, 4, 64, dtype=BF16, device=DEV, requires_grad=True)
    k = torch.zeros(2, 0, 2, 64, dtype=BF16, device=DEV)
    out = sa.causal_attention(q, k, k)
    assert out.shape == q.shape
    assert torch.autograd.grad(out, q, torch.zeros_like(out))[0].shape == q.shape

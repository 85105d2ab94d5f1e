"""rotary_embedding against the definition in 64 bits: layouts, types, part of the head, views, odd sizes, far positions,
packed sequences, gradients, capture into a graph."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _turned(x, positions, f, interleaved, amplitude=1.0, inverse=False):
    """The definition on CPU tensors in 64 bits; also the sum of the magnitudes that a result is made of."""
    x, r = x.double().cpu(), 2 * len(f)
    angle = positions.double().cpu()[..., None] * f.cpu()
    c, s = amplitude * angle.cos()[..., None, :], amplitude * angle.sin()[..., None, :] * (-1 if inverse else 1)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    y, size = x.clone(), x.abs()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = abs(amplitude) * (x[..., a].abs() + x[..., b].abs())
    return y, size


def _check(got, want, size):
    """A result is rounded once to its type (half a step of it); before that cosine and sine are off by at most two steps of
    fp32 (their series and their rounding) plus 2^-24 of angle, the two products and their sum by half a step each: 4 * 2^-23
    of the magnitudes in all."""
    fi = torch.finfo(got.dtype)
    bound = want.abs() * fi.eps / 2 + size * 4 * 2.0 ** -23 + fi.smallest_normal * fi.eps
    assert ((got.double().cpu() - want).abs() <= bound).all(), ((got.double().cpu() - want).abs() / bound).max()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,N,H,HK,D,rot", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 65, 3, 1, 80, 80), (3, 17, 5, 5, 128, 64), (1, 300, 16, 4, 128, 128),
    (2, 33, 2, 0, 96, 32), (1, 7, 3, 2, 36, 12), (1, 5, 2, 1, 33, 22), (1, 9, 1, 1, 256, 256), (2, 1024, 6, 2, 64, 64)])
def test_forward_and_gradient(B, N, H, HK, D, rot, dtype, interleaved):
    g = torch.Generator().manual_seed(B * N + D + rot)
    q = torch.randn(B, N, H, D, generator=g).to(dtype).to(DEV).requires_grad_(True)
    k = torch.randn(B, N, HK, D, generator=g).to(dtype).to(DEV).requires_grad_(True) if HK else None
    f = sa.rotary_frequencies(rot, device=DEV)
    positions = torch.randint(0, 1 << 20, (B, N), generator=g).to(DEV)
    places = torch.arange(N).expand(B, N)
    for given, pos in ((positions, positions), (positions.int(), positions), (None, places)):
        q2, k2 = sa.rotary_embedding(q, k, f, given, interleaved=interleaved, amplitude=1.25)
        dq2 = torch.randn(B, N, H, D, generator=g).to(dtype).to(DEV)
        outs, grads, leaves = [q2], [dq2], [q]
        if HK:
            outs, leaves = [q2, k2], [q, k]
            grads.append(torch.randn(B, N, HK, D, generator=g).to(dtype).to(DEV))
        else:
            assert k2 is None
        found = torch.autograd.grad(outs, leaves, grads)
        for x, y, d, dx in zip(leaves, outs, grads, found):
            _check(y.detach(), *_turned(x.detach(), pos, f, interleaved, 1.25))
            _check(dx, *_turned(d, pos, f, interleaved, 1.25, inverse=True))


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 4, 2, 8, generator=g).to(DEV).requires_grad_(True)
    f = sa.rotary_frequencies(6, device=DEV)
    w = torch.randn(1, 4, 2, 8, generator=g).to(DEV)
    (dq,) = torch.autograd.grad((sa.rotary_embedding(q, None, f)[0] * w).sum(), q)
    step = torch.randn(1, 4, 2, 8, generator=g).to(DEV)
    # linear in q: a difference over a whole step is the derivative, up to the roundings of 64 values of size about 1
    up, down = (((sa.rotary_embedding((q + s * step).detach(), None, f)[0] * w).double().sum()) for s in (0.5, -0.5))
    assert abs((up - down) - (dq * step).double().sum()).item() < 64 * 8 * 2.0 ** -23


def test_views_only_one_gradient_and_other_streams():
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(41, 7, 64, generator=g).bfloat16().to(DEV)
    q, k = fused[:, 1:5], fused[:, 5:6]
    f = sa.rotary_frequencies(32, device=DEV)
    pos = torch.arange(41)
    q2, k2 = sa.rotary_embedding(q, k, f)
    _check(q2, *_turned(q, pos, f, False))
    _check(k2, *_turned(k, pos, f, False))
    odd = torch.randn(5, 3, 70, generator=g).to(DEV)[..., 3:67]                # rows off the 16-byte grid
    _check(sa.rotary_embedding(odd, None, f)[0], *_turned(odd, torch.arange(5), f, False))
    turned = torch.randn(5, 64, 3, generator=g).to(DEV).transpose(1, 2)        # no unit stride: copied
    _check(sa.rotary_embedding(turned, None, f)[0], *_turned(turned, torch.arange(5), f, False))
    kk = k.detach().requires_grad_(True)
    out = sa.rotary_embedding(q, kk, f)
    (dk,) = torch.autograd.grad(out[1], kk, torch.ones_like(out[1]))
    _check(dk, *_turned(torch.ones_like(k), pos, f, False, inverse=True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = sa.rotary_embedding(q, k, f)
    side.synchronize()
    assert torch.equal(again[0], q2) and torch.equal(again[1], k2)


def test_packed_rows():
    g = torch.Generator().manual_seed(4)
    cu = torch.tensor([2, 2, 3, 40, 40, 64], dtype=torch.int32)
    q = torch.randn(70, 2, 64, generator=g).half().to(DEV)
    f = sa.rotary_frequencies(64, device=DEV)
    place = torch.zeros(70, dtype=torch.int64)
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        place[a:b] = torch.arange(b - a)
    _check(sa.rotary_embedding(q, None, f, cu_seqlens=cu.to(DEV), interleaved=True)[0], *_turned(q, place, f, True))
    assert sa.rotary_embedding(q[:0], None, f)[0].shape == (0, 2, 64)


def test_negative_and_largest_positions():
    f = sa.rotary_frequencies(64, device=DEV)
    x = torch.randn(4, 1, 64, generator=torch.Generator().manual_seed(5)).to(DEV)
    pos = torch.tensor([-3, -(1 << 31), (1 << 31) - 1, 1 << 30])
    # an angle of 2^31 radians is formed with 2^-53 of it: 2.4e-7 radians more than the bound of near positions has
    got = sa.rotary_embedding(x, None, f, pos.int().to(DEV))[0].double().cpu()
    want, size = _turned(x, pos, f, False)
    assert ((got - want).abs() <= want.abs() * 2.0 ** -24 + size * (4 * 2.0 ** -23 + 1e-6)).all()


def test_replayed_graph():
    g = torch.Generator().manual_seed(6)
    f = sa.rotary_frequencies(128, device=DEV)
    q, k = (torch.randn(3, 1, h, 128, generator=g).bfloat16().to(DEV) for h in (8, 2))
    pos = torch.zeros(3, 1, dtype=torch.int32, device=DEV)
    sa.rotary_embedding(q, k, f, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = sa.rotary_embedding(q, k, f, pos)
    for i in range(3):
        pos.fill_(100 + i)
        q.copy_(torch.randn(3, 1, 8, 128, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, sa.rotary_embedding(q, k, f, pos)):
            assert torch.equal(a, b)


def test_second_derivatives():
    """The gradient is linear in what comes back, and differentiable in it: turning forth and back again."""
    g = torch.Generator().manual_seed(23)
    q, k = (torch.randn(2, 9, h, 16, generator=g).to(DEV).requires_grad_(True) for h in (3, 1))
    f = sa.rotary_frequencies(8, device=DEV)
    a = [torch.randn(2, 9, h, 16, generator=g).to(DEV).requires_grad_(True) for h in (3, 1)]
    grads = torch.autograd.grad(sa.rotary_embedding(q, k, f), (q, k), a, create_graph=True)
    b = [torch.randn(x.shape, generator=g).to(DEV) for x in grads]
    got = torch.autograd.grad(grads, a, b)
    want = sa.rotary_embedding(*b, f)
    for x, y in zip(got, want):
        assert torch.equal(x, y)

"""tree_attention with a window and first rows that stay visible, and with the weights that cached rows gather, against the
definition in 64 bits: trees, chains and single tokens, pages in any order, windows that end inside a tile or a page, places
that are not used, hidden rows that hold anything, caches beyond 2^31 elements."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def _families(parents):
    """Node lists from the root to each node, None for a place that is not used."""
    out = []
    for i, p in enumerate(parents):
        ok = p == -1 or (0 <= p < i and out[p] is not None)
        out.append(([] if p == -1 else out[p]) + [i] if ok else None)
    return out


def _check(out, q, k, v, parents, kc, vc, lengths, table, scale, window, sinks, rounded, before=None, after=None):
    """Bounds as in causal_util.py: scores off by r, weights by 2 r + w + (n + 16) e, the result rounded to its type; gathered weights
    (never rounded to 16 bits) by 2 r + (n + 16) e of each head's and e of the sum for each of its G + 1 additions."""
    B, T, H, D = q.shape
    HK, dtype = k.shape[2], q.dtype
    G, page = H // HK, kc.shape[1]
    t = torch.finfo(dtype).eps / 2
    w, low = (t, 2.0 ** -25 if dtype == FP16 else 0.0) if rounded else (E, 0.0)
    W = window or 1 << 40
    for b in range(B):
        n = max(0, min(int(lengths[b]), page * (table.shape[1] if table is not None else 1)))
        at = torch.arange(n)
        if table is None:
            there = torch.ones(n, dtype=torch.bool)
            rows = [c[b, :n] for c in (kc, vc)]
        else:
            pages = table[b].long()[at // page]
            there = (pages >= 0) & (pages < kc.shape[0])
            rows = [c[pages[there].to(DEV), (at % page)[there].to(DEV)] for c in (kc, vc)]
        at = at[there]
        family = _families(parents[b].tolist() if parents is not None else list(range(-1, T - 1)))
        for i in range(T):
            if family[i] is None:
                assert out[b, i].count_nonzero() == 0
                continue
            place = n + len(family[i]) - 1
            held = ((place - at < W) | (at < sinks)).to(DEV)
            nodes = [j for d, j in enumerate(family[i]) if place - (n + d) < W or n + d < sinks]
            for h in range(H):
                K, V = (torch.cat((c[held, h // G], new[b, nodes, h // G])).double() for c, new in zip(rows, (k, v)))
                Q = q[b, i, h].double()
                S = K @ Q * scale
                P = torch.softmax(S, 0)
                r = (D + 4) * E * abs(scale) * (K.abs() @ Q.abs()).max()
                want = P @ V
                rel = 2 * r + (len(V) + 16) * E
                bound = (P @ V.abs()) * (rel + w) + low * V.abs().sum(0) + t * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
                far = ((out[b, i, h].double() - want).abs() / bound).max()
                assert far <= 1, (b, i, h, far.item())
                if before is not None:
                    if h % G == 0:
                        sums, off = before[b, h // G].double().clone(), torch.zeros_like(before[b, h // G], dtype=torch.float64)
                    to = torch.cat((at[held.cpu()], torch.tensor([n]))).to(DEV)
                    real = to < sums.numel()
                    capacity = page * (table.shape[1] if table is not None else 1)
                    real &= to < capacity
                    sums[to[real]] += P[real]
                    off[to[real]] += P[real] * rel
                    if h % G == G - 1:
                        off += (G + 1) * E * sums.abs() + 2.0 ** -140
                        far = ((after[b, h // G].double() - sums).abs() / off).max()
                        assert far <= 1, ("weights", b, h // G, far.item())
                        touched = torch.zeros(sums.numel(), dtype=torch.bool, device=DEV)
                        touched[to[real]] = True
                        assert torch.equal(after[b, h // G][~touched], before[b, h // G][~touched])


def _random_parents(B, T, g, holes=True):
    rows = []
    for b in range(B):
        n = T if b == 0 or not holes else int(torch.randint(0, T + 1, (), generator=g))
        up = [-1] + [int(torch.randint(max(-1, i - 3), i, (), generator=g)) for i in range(1, n)]
        rows.append((up + [-2] * T)[:n] + [-2] * (T - n))
    return torch.tensor(rows, dtype=torch.int32)


def _case(B, T, H, HK, D, page, width, dtype, seed, paged=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    q, k, v = make(B, T, H, D) * std, make(B, T, HK, D), make(B, T, HK, D)
    pages = B * width + 3 if paged else B
    kc, vc = (make(pages, page if paged else page * width, HK, D) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int() if paged else None
    lengths = torch.randint(0, page * width + 1, (B,), generator=g).int()
    lengths[0] = page * width
    return q, k, v, _random_parents(B, T, g), kc, vc, lengths, table


def _run(q, k, v, parents, kc, vc, lengths, table, window, sinks, flags=0, scale=None, weights=None):
    up = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    return sa.tree_attention(q, k, v, up(parents), kc, vc, up(lengths), up(table), scale, flags, window, sinks, weights)


SHAPES = [(3, 1, 4, 2, 128, 16, 20), (2, 1, 16, 4, 64, 64, 9), (1, 1, 8, 1, 80, 5, 77), (2, 7, 4, 4, 64, 16, 30), (3, 23, 8, 2, 128, 32, 12),
          (2, 64, 4, 1, 128, 16, 25), (2, 33, 2, 2, 32, 100, 3), (1, 64, 8, 2, 64, 48, 7), (4, 5, 6, 2, 256, 16, 9), (2, 9, 3, 1, 33, 7, 20), (2, 1, 70, 1, 128, 16, 24)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 3), (64, 0), (100, 1), (65, 70), (200, 40), (10000, 3)])
@pytest.mark.parametrize("dtype,flags", [(BF16, 0), (FP16, 0), (FP32, 0), (BF16, _lib.FLAG_FORCE_GENERIC)])
@pytest.mark.parametrize("B,T,H,HK,D,page,width", SHAPES)
def test_windows(B, T, H, HK, D, page, width, dtype, flags, window, sinks):
    q, k, v, parents, kc, vc, lengths, table = _case(B, T, H, HK, D, page, width, dtype, B + T + D)
    for b in range(1, B):                                   # some sequences shorter than the window, or empty
        lengths[b] = int(lengths[b]) % (window + sinks + 9) if b % 2 else lengths[b]
    out = _run(q, k, v, parents, kc, vc, lengths, table, window, sinks, flags)
    _check(out, q, k, v, parents, kc, vc, lengths, table, D ** -0.5, window, sinks, dtype != FP32 and not flags)


@pytest.mark.parametrize("dtype,flags", [(BF16, 0), (FP16, 0), (FP32, 0), (FP16, _lib.FLAG_FORCE_GENERIC)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 4), (1, 0)])
@pytest.mark.parametrize("B,H,HK,D,page,width,paged", [(3, 4, 2, 128, 16, 20, True), (2, 16, 4, 64, 64, 9, True), (1, 8, 1, 80, 500, 1, False), (4, 2, 2, 32, 33, 5, True),
                                                       (2, 70, 1, 128, 16, 24, True), (2, 3, 1, 200, 16, 6, True), (1, 4, 4, 128, 16, 400, True)])
def test_weights(B, H, HK, D, page, width, paged, window, sinks, dtype, flags):
    q, k, v, _, kc, vc, lengths, table = _case(B, 1, H, HK, D, page, width, dtype, B + H + D, paged)
    if B > 2:
        lengths[1] = 0
    lengths[B - 1] = page * width - 7
    extra = 5 if B == 2 else 0                              # (more places than the cache has)
    before = torch.rand(B, HK, page * width + extra, generator=torch.Generator().manual_seed(3)).to(DEV)
    after = before.clone()
    out = _run(q, k, v, None, kc, vc, lengths, table, window, sinks, flags, weights=after)
    _check(out, q, k, v, None, kc, vc, lengths, table, D ** -0.5, window, sinks, dtype != FP32 and not flags, before, after)
    assert torch.equal(out, _run(q, k, v, None, kc, vc, lengths, table, window, sinks, flags, weights=torch.zeros_like(before)))
    if table is not None:                                   # pages that are none of the cache's: their rows are not there
        table[0, ::3] = -1
        after = before.clone()
        out = _run(q, k, v, None, kc, vc, lengths, table, window, sinks, flags, weights=after)
        _check(out, q, k, v, None, kc, vc, lengths, table, D ** -0.5, window, sinks, dtype != FP32 and not flags, before, after)


def test_an_unused_place_gathers_nothing():
    q, k, v, _, kc, vc, lengths, table = _case(2, 1, 4, 2, 64, 16, 8, BF16, 5)
    weights = torch.rand(2, 2, 128, device=DEV)
    before = weights.clone()
    out = _run(q, k, v, torch.tensor([[-2], [-1]], dtype=torch.int32), kc, vc, lengths, table, None, 0, weights=weights)
    assert out[0].count_nonzero() == 0 and torch.equal(weights[0], before[0]) and not torch.equal(weights[1], before[1])


def test_scales_of_any_sign():
    for scale in (-0.2, 0.0, 0.7):
        q, k, v, _, kc, vc, lengths, table = _case(2, 1, 4, 2, 64, 16, 8, BF16, 6)
        table[0, 2] = 999
        before = torch.rand(2, 2, 128, device=DEV)
        after = before.clone()
        out = _run(q, k, v, None, kc, vc, lengths, table, 60, 3, scale=scale, weights=after)
        _check(out, q, k, v, None, kc, vc, lengths, table, scale, 60, 3, True, before, after)


@pytest.mark.parametrize("dtype,flags", [(BF16, 0), (FP16, 0), (FP32, 0)])
@pytest.mark.parametrize("T,H,HK,D", [(1, 4, 2, 128), (6, 4, 2, 64), (40, 8, 2, 128), (3, 2, 1, 256)])
def test_hidden_rows_may_hold_anything(T, H, HK, D, dtype, flags):
    """NaN and infinities in rows out of the window, behind the sequence and in nodes that nobody sees change nothing."""
    window, sinks, n = 70, 5, 333
    q, k, v, parents, kc, vc, lengths, table = _case(1, T, H, HK, D, 16, 24, dtype, 8)
    lengths[0] = n
    parents = _random_parents(1, T, torch.Generator().manual_seed(1), holes=False)
    want = _run(q, k, v, parents, kc, vc, lengths, table, window, sinks, flags)

    def same(a, b):
        # Other sums in the tile that holds such a row: 2 (n + 16) e of magnitudes below 16, then a rounding of each.  In 16 bits a
        # workgroup may sweep a second time for a row that does see it: the weights, whose sum is 1, are then rounded against another
        # reference point, half a step (eps / 2) of each on either side, which the values (all below 8) carry on
        weights = torch.finfo(dtype).eps * 8 if dtype != FP32 else 0.0
        return ((a.double() - b.double()).abs() <= torch.finfo(dtype).eps * b.double().abs() + 2 * (n + 16) * E * 16 + weights).all()

    for bad in (math.nan, math.inf, -math.inf):
        k2, v2 = kc.clone(), vc.clone()
        for r in [*range(sinks, n - window + 1), *range(n, 24 * 16)]:      # what no node sees
            k2[table[0, r // 16], r % 16, :, 1], v2[table[0, r // 16], r % 16, :, 2] = bad, bad
        assert same(_run(q, k, v, parents, k2, v2, lengths, table, window, sinks, flags), want)
        if T > 1:                                           # what the deepest node does not see, but others do
            depth = [len(f) - 1 for f in _families(parents[0].tolist())]
            far = [i for i, d in enumerate(depth) if d >= 2]
            k2, v2 = kc.clone(), vc.clone()
            r = n - window + 2
            k2[table[0, r // 16], r % 16, :, 1], v2[table[0, r // 16], r % 16, :, 2] = bad, bad
            out = _run(q, k, v, parents, k2, v2, lengths, table, window, sinks, flags)
            assert same(out[:, far], want[:, far])


def test_long_caches():
    """Offsets beyond 2^31 elements, a window at the far end of a cache."""
    n, HK, D, page = 9_000_000, 2, 128, 4096
    pages = n // page + 1
    kc, vc = (torch.empty(pages, page, HK, D, dtype=BF16, device=DEV) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(1)
    for t in (kc, vc):
        t[-2:].normal_(generator=g)
        t[:1].normal_(generator=g)
    q, k, v = (torch.randn(1, 2, h, D, generator=g, device=DEV).to(BF16) for h in (4, HK, HK))
    table = torch.arange(pages, device=DEV, dtype=torch.int32)[None]
    for lengths in (n, n - 777):
        held = torch.tensor([lengths], dtype=torch.int32, device=DEV)
        out = sa.tree_attention(q, k, v, None, kc, vc, held, table, window=600, sinks=4)
        rows = [torch.cat((t.flatten(0, 1)[:4], t.flatten(0, 1)[lengths - 599:lengths], new[0])) for t, new in ((kc, k), (vc, v))]
        for h in range(4):
            S = q[0, :, h].double() @ rows[0][:, h // 2].double().T * D ** -0.5
            S[0, -1] = -math.inf                            # node 0 does not see node 1, node 1 not the window's first row
            S[1, 4] = -math.inf
            want = torch.softmax(S, 1) @ rows[1][:, h // 2].double()
            assert ((out[0, :, h].double() - want).abs() <= 2.0 ** -7 * (1 + want.abs())).all()


def test_graphs_follow_lengths_and_windows_slide():
    q, k, v, _, kc, vc, _, table = _case(2, 1, 8, 2, 128, 16, 40, BF16, 12)
    lengths, table = torch.tensor([300, 10], dtype=torch.int32, device=DEV), table.to(DEV)
    weights = torch.zeros(2, 2, 640, device=DEV)
    sa.tree_attention(q, k, v, None, kc, vc, lengths, table, window=100, sinks=4, weights=weights)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = sa.tree_attention(q, k, v, None, kc, vc, lengths, table, window=100, sinks=4, weights=weights)
    for step in range(4):
        lengths += 37
        weights.zero_()
        graph.replay()
        torch.cuda.synchronize()
        fresh = torch.zeros_like(weights)
        assert torch.equal(out, sa.tree_attention(q, k, v, None, kc, vc, lengths, table, window=100, sinks=4, weights=fresh))
        assert torch.equal(weights, fresh)
        # one token's weights are G of them
        assert (weights.sum(2) - 4).abs().max() < 1e-4

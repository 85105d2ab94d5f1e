"""cache_evict against the definition on the CPU, row by row: pages in any order, equal weights, NaN and infinities among them, one choice
for all heads, odd sizes, lengths outside of the cache, caches beyond 2^31 elements, graphs; and the operators together."""
import math

import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _chosen(w, n, keep, first, recent):
    """Places of one head that stay."""
    if n <= keep:
        return list(range(n))
    x = [-math.inf if math.isnan(v) else v for v in w[:n].tolist()]
    nan = [math.isnan(v) for v in w[:n].tolist()]
    free = sorted(range(first, n - recent), key=lambda i: (nan[i], -x[i], i))
    return sorted(list(range(first)) + free[:keep - first - recent] + list(range(n - recent, n)))


def _expect(kc, vc, w, lengths, table, keep, first, recent):
    kc, vc, w = kc.cpu().clone(), vc.cpu().clone(), w.cpu()
    B, heads, places = w.shape
    page, HK = kc.shape[1], kc.shape[2]
    capacity = page * (table.shape[1] if table is not None else 1)
    kept, left = torch.full((B, heads, keep), -1, dtype=torch.int32), torch.zeros(B, heads, places)
    old = kc.clone(), vc.clone()
    for b in range(B):
        n = max(0, min(int(lengths[b]), capacity))
        for hk in range(HK):
            h = hk if heads > 1 else 0
            stay = _chosen(w[b, h], n, keep, first, recent)
            kept[b, h, :len(stay)] = torch.tensor(stay, dtype=torch.int32)
            left[b, h, :len(stay)] = w[b, h, stay]
            if table is None:
                kc[b, :len(stay), hk], vc[b, :len(stay), hk] = old[0][b, stay, hk], old[1][b, stay, hk]
                continue
            for i, r in enumerate(stay):
                src, dst = ((b, x) if table is None else (int(table[b, x // page]), x % page) for x in (r, i))
                if r != i and 0 <= src[0] < kc.shape[0] and 0 <= dst[0] < kc.shape[0]:
                    kc[dst[0], dst[1], hk], vc[dst[0], dst[1], hk] = old[0][src[0], src[1], hk], old[1][src[0], src[1], hk]
    return kept, left, kc, vc


def _same(a, b):
    return torch.equal(a.nan_to_num(nan=-123.0), b.nan_to_num(nan=-123.0))


def _run(kc, vc, w, lengths, table, keep, first, recent):
    kc, vc = kc.clone(), vc.clone()
    kept, left = sa.cache_evict(kc, vc, w, lengths.to(DEV), keep, first, recent, None if table is None else table.to(DEV))
    return kept, left, kc, vc


def _case(B, HK, heads, D, page, width, dtype, seed, paged, extra=0):
    g = torch.Generator().manual_seed(seed)
    pages = B * width + 2 if paged else B
    kc, vc = (torch.randn(pages, page if paged else page * width, HK, D, generator=g).to(dtype).to(DEV) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int() if paged else None
    w = torch.randn(B, heads, page * width + extra, generator=g).mul_(2).exp_()
    w[torch.rand(w.shape, generator=g) < 0.2] = 0.0
    lengths = torch.randint(page * width // 2, page * width + 1, (B,), generator=g).int()
    return kc, vc, w.to(DEV), lengths, table


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("B,HK,heads,D,page,width,keep,first,recent,paged,extra", [
    (1, 1, 1, 64, 1, 7, 3, 0, 0, True, 0), (2, 2, 2, 128, 16, 20, 100, 4, 30, True, 0), (3, 4, 4, 80, 16, 9, 1, 1, 0, True, 3), (2, 2, 1, 32, 33, 5, 77, 0, 10, True, 0),
    (2, 3, 3, 33, 100, 7, 333, 5, 200, False, 0), (1, 8, 8, 128, 64, 40, 600, 0, 0, True, 0), (4, 2, 2, 128, 16, 60, 959, 4, 100, True, 0), (2, 1, 1, 1, 50, 30, 700, 0, 699, False, 0),
    (1, 2, 2, 64, 512, 11, 2000, 10, 1990, True, 0), (2, 4, 1, 256, 16, 30, 333, 2, 3, True, 8), (1, 2, 2, 64, 16, 300, 4500, 0, 1, True, 0)])
def test_rows_that_stay(B, HK, heads, D, page, width, keep, first, recent, paged, extra, dtype):
    kc, vc, w, lengths, table = _case(B, HK, heads, D, page, width, dtype, B + D + width, paged, extra)
    if B > 1:
        lengths[B - 1] = page * width
    if B > 2:
        lengths[0], lengths[1] = 0, min(keep, page * width)
    got = _run(kc, vc, w, lengths, table, keep, first, recent)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, _expect(kc, vc, w, lengths, table, keep, first, recent)))


@pytest.mark.parametrize("values", ["equal", "zeros", "signs", "odd", "close"])
def test_weights_of_any_kind(values):
    kc, vc, w, lengths, table = _case(2, 2, 2, 64, 16, 100, BF16, 3, True)
    g = torch.Generator().manual_seed(4)
    if values == "equal":
        w = torch.full_like(w, 0.25)
    elif values == "zeros":
        w = torch.zeros_like(w)
        w[..., ::2] *= -1.0                                 # (-0 is 0)
    elif values == "signs":
        w = (torch.randint(-3, 4, w.shape, generator=g).float()).to(DEV)
    elif values == "odd":
        pick = torch.randint(0, 5, w.shape, generator=g).to(DEV)
        for i, bad in enumerate((math.nan, math.inf, -math.inf, -math.nan)):
            w[pick == i] = bad
    else:                                                   # neighbouring numbers
        w = (1.0 + torch.randint(0, 300, w.shape, generator=g).float() * 2.0 ** -23).to(DEV)
    for keep, first, recent in ((500, 4, 100), (1400, 0, 0), (3, 1, 1)):
        got = _run(kc, vc, w, lengths, table, keep, first, recent)
        want = _expect(kc, vc, w, lengths, table, keep, first, recent)
        assert torch.equal(got[0].cpu(), want[0]) and _same(got[1].cpu(), want[1]) and all(torch.equal(a.cpu(), b) for a, b in zip(got[2:], want[2:]))


@pytest.mark.parametrize("values", ["drawn", "equal", "few"])
@pytest.mark.parametrize("heads,paged", [(2, True), (1, True), (2, False)])
def test_workgroups_that_share_a_head(heads, paged, values):
    """Caches of 32768 rows on: the weights that are equal, the first and the last rows fall into any of the parts, or into none."""
    kc, vc, w, lengths, table = _case(6, 2, heads, 8, 300, 110, FP16, 7, paged, 1)
    g = torch.Generator().manual_seed(8)
    if values == "equal":
        w = torch.ones_like(w)
    elif values == "few":
        w = torch.randint(0, 3, w.shape, generator=g).float().to(DEV)
    lengths = torch.tensor([33000, 32768, 4097, 100, 0, 17000], dtype=torch.int32)
    for keep, first, recent in ((8300, 4, 4000), (90, 0, 50), (32999, 20000, 10), (16500, 0, 16500)):
        got = _run(kc, vc, w, lengths, table, keep, first, recent)
        want = _expect(kc, vc, w, lengths, table, keep, first, recent)
        assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))


def test_pages_and_lengths_outside_of_the_cache():
    kc, vc, w, lengths, table = _case(4, 2, 2, 64, 16, 30, BF16, 7, True)
    table[0, ::4], table[1, 5] = -1, 10_000
    lengths[:] = torch.tensor([480, 400, 9999, -5])
    got = _run(kc, vc, w, lengths, table, 150, 3, 40)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, _expect(kc, vc, w, lengths, table, 150, 3, 40)))


def test_views_of_caches_and_weights():
    """Heads and rows of a larger tensor, off the 16-byte grid; what stands beside them is left as it is."""
    g = torch.Generator().manual_seed(1)
    for off in (0, 1):
        whole = [torch.randn(3, 500, 4, 72, generator=g).to(BF16).to(DEV) for _ in range(2)]
        kept_whole = [t.clone() for t in whole]
        views = [t[:, :, 1:3, off:off + 64] for t in whole]
        w = torch.rand(3, 6, 510, generator=g).to(DEV)[:, 2:4]
        lengths = torch.tensor([500, 300, 420], dtype=torch.int32)
        want = _expect(*[v.contiguous() for v in views], w, lengths, None, 200, 1, 50)
        kept, left = sa.cache_evict(*views, w, lengths.to(DEV), 200, 1, 50)
        assert torch.equal(kept.cpu(), want[0]) and torch.equal(left.cpu(), want[1])
        for t, old, v in zip(whole, kept_whole, want[2:]):
            old[:, :, 1:3, off:off + 64] = v.to(DEV)
            assert torch.equal(t, old)


def test_long_caches():
    """Many steps of the movers, and offsets beyond 2^31 elements."""
    B, HK, D, page = 2, 2, 128, 4096
    pages = 9000                                            # 9.4e9 elements
    kc, vc = (torch.empty(pages, page, HK, D, dtype=BF16, device=DEV) for _ in range(2))
    width = 30
    table = torch.stack((torch.arange(pages - width, pages), torch.arange(0, 2 * width, 2))).int()
    g = torch.Generator(device=DEV).manual_seed(1)
    for t in (kc, vc):
        for p in table.flatten().tolist():
            t[p].normal_(generator=g)
    w = torch.rand(B, HK, page * width, device=DEV, generator=g)
    lengths = torch.tensor([page * width, page * width - 1000], dtype=torch.int32)
    old = [torch.stack([t[table[b].long()].flatten(0, 1) for b in range(B)]) for t in (kc, vc)]
    keep, first, recent = 70_000, 4, 5000
    kept, left = sa.cache_evict(kc, vc, w, lengths.to(DEV), keep, first, recent, table.to(DEV))
    for b in range(B):
        n = int(lengths[b])
        place = torch.arange(page * width, device=DEV)
        rank = w[b].masked_fill((place < first) | (place >= n - recent), math.inf).masked_fill(place >= n, -math.inf)
        want = rank.sort(dim=-1, descending=True, stable=True)[1][:, :keep].sort(-1)[0]
        assert torch.equal(kept[b].long(), want) and torch.equal(left[b, :, :keep], w[b].gather(1, want)) and left[b, :, keep:].count_nonzero() == 0
        for t, o in zip((kc, vc), old):
            now = t[table[b].long()].flatten(0, 1)
            assert torch.equal(now[keep:], o[b, keep:])
            for h in range(HK):
                assert torch.equal(now[:keep, h], o[b, want[h], h])


def test_graphs():
    kc, vc, w, lengths, table = _case(2, 2, 2, 128, 16, 40, BF16, 9, True)
    table, held = table.to(DEV), lengths.to(DEV)
    sa.cache_evict(kc.clone(), vc.clone(), w, held, 200, 2, 30, table)
    static = [t.clone() for t in (kc, vc, w)]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept, left = sa.cache_evict(*static, held, 200, 2, 30, table)
    for seed in (1, 2, 3):
        kc2, vc2, w2, lengths2, _ = _case(2, 2, 2, 128, 16, 40, BF16, 9 + seed, True)
        for t, x in zip((*static, held), (kc2, vc2, w2, lengths2)):
            t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want = _expect(kc2, vc2, w2, lengths2, table.cpu(), 200, 2, 30)
        assert all(torch.equal(a.cpu(), b) for a, b in zip((kept, left, *static[:2]), want))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_the_operators_together(dtype):
    """Prompts into a cache, what their keys were worth, decoding steps that add to it, an eviction, further steps: the last
    steps' outputs are attention over the rows that stayed."""
    g = torch.Generator().manual_seed(17)
    H, HK, D, page, width, keep, window, sinks = 4, 2, 64, 16, 30, 160, 100, 4
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    ends = [0, 300, 300, 420]
    B, T = len(ends) - 1, ends[-1]
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    table = torch.randperm(B * width, generator=g).view(B, width).int().to(DEV)
    kc, vc = make(B * width, page, HK, D), make(B * width, page, HK, D)
    weights, lengths = torch.zeros(B, HK, page * width, device=DEV), torch.zeros(B, dtype=torch.int32, device=DEV)
    f = sa.rotary_frequencies(D, device=DEV)
    q, k = sa.rotary_embedding(make(T, H, D), make(T, HK, D), f, cu_seqlens=cu)
    v = make(T, HK, D)
    out, lse = sa.causal_attention_forward(q, k, v, cu, window=window, sinks=sinks)
    sa.key_weights(q, k, lse, cu, window=window, sinks=sinks, weights=weights, lengths=lengths)
    sa.cache_append(k, v, kc, vc, lengths, table, cu_seqlens=cu)
    lengths += cu.diff()
    # the last prompt token again, as a decoding step, is what the prompt's attention gave
    last = torch.tensor([299, 419], device=DEV)
    again = sa.tree_attention(q[last][:, None], k[last][:, None], v[last][:, None], None, kc, vc, lengths[[0, 2]] - 1, table[[0, 2]], window=window, sinks=sinks)
    # (two roundings of the result, and of the weights, whose sum is 1, over values below 8)
    t = torch.finfo(dtype).eps
    assert ((again[:, 0] - out[last]).double().abs() <= t * out[last].double().abs() + (8 * t if dtype != FP32 else 2e-5)).all()
    assert ((weights.sum(2) - cu.diff()[:, None] * (H // HK)).abs() <= 1e-3).all()
    position = lengths.clone()
    for step in range(6):
        qs, ks = sa.rotary_embedding(make(B, 1, H, D), make(B, 1, HK, D), f, positions=position[:, None])
        vs = make(B, 1, HK, D)
        sa.tree_attention(qs, ks, vs, None, kc, vc, lengths, table, weights=weights)
        sa.cache_append(ks, vs, kc, vc, lengths, table)
        lengths += 1
        position += 1
        if step == 2:
            rows = [torch.stack([t[table[b].long()].flatten(0, 1) for b in range(B)]) for t in (kc, vc)]
            kept, weights = sa.cache_evict(kc, vc, weights, lengths, keep, first=sinks, recent=32, page_table=table)
            old, lengths = lengths, lengths.clamp(max=keep)
            for t, o in zip((kc, vc), rows):
                for b in range(B):
                    now, n = t[table[b].long()].flatten(0, 1), int(lengths[b])
                    for h in range(HK):
                        assert torch.equal(now[:n, h], o[b, kept[b, h, :n].long(), h])
            assert (kept[1, :, 3:] == -1).all() and (old - lengths).tolist() == [303 - keep, 0, 0]
    assert lengths.tolist() == [keep + 3, 6, 126] and position.tolist() == [306, 6, 126]
    qs, ks, vs = make(B, 1, H, D), make(B, 1, HK, D), make(B, 1, HK, D)
    out = sa.tree_attention(qs, ks, vs, None, kc, vc, lengths, table)
    for b in range(B):
        n = int(lengths[b])
        for h in range(H):
            K, V = (torch.cat((t[table[b].long()].flatten(0, 1)[:n, h // 2], x[b, :, h // 2])).double() for t, x in ((kc, ks), (vc, vs)))
            want = torch.softmax(K @ qs[b, 0, h].double() * D ** -0.5, 0) @ V
            assert ((out[b, 0, h].double() - want).abs() <= (t_ := torch.finfo(dtype).eps) * want.abs() + (8 * t_ if dtype != FP32 else 2e-5)).all()

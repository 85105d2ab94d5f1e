"""tree_attention against the definition in 64 bits: trees, chains and single tokens, pages in any order, lengths that end
inside a tile or a page, places that are not used, whatever lies behind a sequence's rows, caches beyond 2^31 elements."""
import math

import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
E = 2.0 ** -24


def _ancestors(parents):
    """[T, T] bool of one sequence, on the CPU: row i is empty for a place that is not used."""
    T = len(parents)
    seen = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        j, row = i, torch.zeros(T, dtype=torch.bool)
        while 0 <= j < T:
            row[j] = True
            up = parents[j]
            if up == -1:
                seen[i] = row
                break
            if not -1 <= up < j:
                break
            j = up
    return seen


def _check(out, q, k, v, parents, kc, vc, lengths, table, scale):
    """Bounds as in causal_util.py: scores off by r, weights by 2 r + w + (n + 16) e, the result rounded to its type."""
    B, T, H, D = q.shape
    HK, dtype = k.shape[2], q.dtype
    G, page = H // HK, kc.shape[1]
    t = torch.finfo(dtype).eps / 2
    w, low = (E, 0.0) if dtype == FP32 else (t, 2.0 ** -25 if dtype == FP16 else 0.0)
    for b in range(B):
        n = max(0, min(int(lengths[b]), page * (table.shape[1] if table is not None else 1)))
        if table is None:
            rows = [c[b, :n] for c in (kc, vc)]
        else:
            at = torch.arange(n)
            pages = table[b].long()[at // page]
            there = (pages >= 0) & (pages < kc.shape[0])
            rows = [c[pages[there].to(DEV), (at % page)[there].to(DEV)] for c in (kc, vc)]
        n = rows[0].shape[0]
        seen = _ancestors(parents[b].tolist() if parents is not None else list(range(-1, T - 1)))
        mask = torch.cat((seen.any(1, keepdim=True).expand(T, n), seen), 1).to(DEV)
        keep = seen.any(0)
        for h in range(H):
            # drafted rows that nobody sees are left out: they may hold anything
            cols = torch.cat((torch.ones(n, dtype=torch.bool), keep)).to(DEV)
            K, V = (torch.cat((c[:, h // G], new[b, :, h // G])).double()[cols] for c, new in zip(rows, (k, v)))
            M, used = mask[:, cols], mask.any(1)
            assert out[b, ~used, h].count_nonzero() == 0
            if not used.any():
                continue
            Q = q[b, used, h].double()
            S = (Q @ K.T * scale).masked_fill(~M[used], -math.inf)
            P = torch.softmax(S, 1)
            r = ((D + 4) * E * abs(scale) * (Q.abs() @ K.abs().T)).masked_fill(~M[used], 0).amax(1, keepdim=True)
            want = P @ V
            bound = (P @ V.abs()) * (2 * r + w + (len(V) + 16) * E) + low * (M[used].double() @ V.abs()) + t * want.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            far = ((out[b, used, h].double() - want).abs() / bound).max()
            assert far <= 1, (b, h, far.item())


def _random_parents(B, T, g, holes=True):
    rows = []
    for b in range(B):
        n = T if b == 0 or not holes else int(torch.randint(0, T + 1, (), generator=g))
        up = [-1] + [int(torch.randint(-1, i, (), generator=g)) for i in range(1, n)]
        rows.append((up + [-2] * T)[:n] + [-2] * (T - n))
    return torch.tensor(rows, dtype=torch.int32)


def _case(B, T, H, HK, D, page, width, dtype, seed, paged=True, std=1.0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)
    q, k, v = make(B, T, H, D) * std, make(B, T, HK, D), make(B, T, HK, D)
    pages = B * width + 3 if paged else B
    kc, vc = (make(pages, page if paged else page * width, HK, D) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int() if paged else None
    lengths = torch.randint(0, page * width + 1, (B,), generator=g).int()
    return q, k, v, _random_parents(B, T, g), kc, vc, lengths, table


def _run(q, k, v, parents, kc, vc, lengths, table, scale=None):
    on = lambda t: t.to(DEV) if t is not None else None
    return sa.tree_attention(q, k, v, on(parents), kc, vc, on(lengths), on(table), scale)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("B,T,H,HK,D,page,width", [
    (1, 1, 1, 1, 64, 1, 1), (3, 1, 8, 2, 128, 16, 9), (2, 5, 4, 4, 64, 64, 5), (4, 64, 2, 1, 128, 16, 20), (2, 33, 6, 2, 80, 32, 8),
    (1, 17, 16, 2, 128, 7, 31), (2, 3, 3, 1, 33, 16, 12), (2, 9, 2, 2, 256, 16, 10), (1, 2, 8, 1, 32, 256, 9), (5, 12, 12, 4, 64, 128, 20), (2, 1, 5, 1, 8, 3, 40)])
def test_trees(B, T, H, HK, D, page, width, dtype, paged):
    x = _case(B, T, H, HK, D, page, width, dtype, B * T + D + page, paged)
    _check(_run(*x), *x, D ** -0.5)
    lengths = x[6]
    for n in (0, 1, 31, 32, 33, page * width):                 # nothing, one row, the ends of tiles, everything
        lengths.fill_(min(n, page * width))
        _check(_run(*x), *x, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("B,T,H,HK,D,page,width", [
    (1, 64, 16, 2, 128, 16, 260), (2, 48, 16, 4, 128, 64, 40), (1, 33, 4, 2, 64, 7, 300), (3, 64, 4, 2, 64, 32, 30), (2, 20, 20, 1, 80, 3, 700), (1, 64, 3, 1, 128, 5, 999)])
def test_many_rows(B, T, H, HK, D, page, width, dtype):
    """More than 64 rows per key head: the wavefronts of a workgroup divide the rows and share the keys."""
    x = _case(B, T, H, HK, D, page, width, dtype, T + D + page)
    _check(_run(*x), *x, D ** -0.5)
    lengths, table, kc = x[6], x[7], x[4]
    for n in (0, 63, 64, 65, page * width):
        lengths.fill_(min(n, page * width))
        _check(_run(*x), *x, D ** -0.5)
    table[0, width // 2], table[-1, 0] = -1, kc.shape[0]       # pages that are none
    _check(_run(*x), *x, D ** -0.5)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,H,D", [(64, 4, 64), (64, 4, 128), (40, 2, 128), (3, 2, 64)])
def test_later_keys_far_above_the_first(T, H, D, dtype):
    x = _case(1, T, H, 1, D, 64, 40, dtype, 61, std=8.0)
    x[6].fill_(64 * 40)
    x[4][x[7][0, 0].long()] *= 0.01
    _check(_run(*x, 0.5), *x, 0.5)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_long_tables(dtype):
    """One long cache shared by 64 workgroups; a table longer than a workgroup keeps in LDS."""
    x = _case(1, 2, 4, 1, 64, 16, 2100, dtype, 71)
    x[6].fill_(16 * 2100 - 5)
    _check(_run(*x), *x, 0.125)
    x = _case(64, 1, 8, 4, 64, 1, 4500, dtype, 73)
    out = _run(*x)
    part = lambda t, b: t[b:b + 1]
    for b in (0, 40, 63):
        _check(part(out, b), *(part(t, b) for t in x[:4]), x[4], x[5], part(x[6], b), part(x[7], b), 0.125)


def test_shares_of_a_long_table_of_single_rows():
    """Full caches behind pages of one row: shares that are longer than an eighth of the table."""
    x = _case(2, 64, 32, 16, 64, 1, 30000, BF16, 79)
    x[6].fill_(30000)
    _check(_run(*x), *x, 0.125)
    x[6][1] = 31
    _check(_run(*x), *x, 0.125)


@pytest.mark.parametrize("B,T,cap", [(4, 12, 65536), (32, 16, 2048), (3, 9, 40000)])
def test_few_rows_over_many_keys(B, T, cap):
    x = _case(B, T, 16, 4, 128, 64, cap // 64, BF16, 83)
    x[6].fill_(cap - 9)
    x[6][0] = 0
    x[6][B // 2] = cap // 3
    out = _run(*x)
    for b in (0, B // 2, B - 1):
        part = lambda t: t[b:b + 1]
        _check(part(out), *(part(t) for t in x[:4]), x[4], x[5], part(x[6]), part(x[7]), 128 ** -0.5)


def test_chain_and_bad_parents():
    q, k, v, _, kc, vc, lengths, table = _case(2, 7, 4, 2, 64, 16, 6, BF16, 3)
    chain = torch.arange(-1, 6, dtype=torch.int32).expand(2, 7).contiguous()
    assert torch.equal(_run(q, k, v, None, kc, vc, lengths, table), _run(q, k, v, chain, kc, vc, lengths, table))
    # a parent that is itself, comes later, or is no number of a node: the place and what hangs on it are not used
    odd = torch.tensor([[-1, 1, 0, 5, 2, -7, 9], [-2, 0, -1, 2, 1, 3, 100]], dtype=torch.int32)
    x = (q, k, v, odd, kc, vc, lengths, table)
    _check(_run(*x), *x, 0.125)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [64, 128])
def test_what_is_not_there_may_hold_anything(dtype, D):
    q, k, v, parents, kc, vc, lengths, table = _case(3, 6, 4, 2, D, 16, 12, dtype, 9)
    lengths = torch.tensor([0, 75, 192]).int()
    parents = torch.tensor([[-1, 0, 0, 1, -2, -2], [-2] * 6, [-1, -1, 1, 2, 3, -1]], dtype=torch.int32)
    table[1, 2] = -1                                            # no page: rows 32 .. 47 are not there
    table[2, 5] = kc.shape[0]
    want = _run(q, k, v, parents, kc, vc, lengths, table)
    _check(want, q, k, v, parents, kc, vc, lengths, table, D ** -0.5)

    def same(a, b):
        # 200 terms of magnitude 5 at most in another order, then one rounding each
        return ((a.double() - b.double()).abs() <= torch.finfo(dtype).eps * b.double().abs() + 2 * 216 * E * 5).all()

    for bad in (math.nan, math.inf):
        k2, v2, kc2, vc2 = (t.clone() for t in (k, v, kc, vc))
        for t in (k2, v2):
            t[0, 4:], t[1] = bad, bad
        for c in (kc2, vc2):
            held = torch.zeros(c.shape[:2], dtype=torch.bool)
            for b in range(3):
                for r in range(int(lengths[b])):
                    p = int(table[b, r // 16])
                    if 0 <= p < c.shape[0]:
                        held[p, r % 16] = True
            c[~held.to(DEV)] = bad
        assert same(_run(q, k2, v2, parents, kc2, vc2, lengths, table), want)
        # a drafted node with such a value reaches its descendants only
        v3 = v.clone()
        v3[2, 2] = bad
        got = _run(q, k, v3, parents, kc, vc, lengths, table)
        assert same(got[2, [0, 1, 5]], want[2, [0, 1, 5]]) and not torch.isfinite(got[2, 2:5].float()).any()
    lengths.fill_(-5)
    assert torch.isfinite(_run(q, k, v, parents, kc, vc, lengths, table).float()).all()
    lengths.fill_(1 << 30)                                      # more than the table holds: all that it holds
    x = (q, k, v, parents, kc, vc, lengths, table)
    _check(_run(*x), *x, D ** -0.5)


def test_scales_and_large_scores():
    x = _case(2, 4, 4, 1, 64, 16, 40, BF16, 15, std=8.0)
    for scale in (0.0, -0.125, 1.0):
        _check(_run(*x, scale), *x, scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_views(dtype):
    q, k, v, parents, kc, vc, lengths, table = _case(2, 5, 4, 2, 64, 16, 8, dtype, 21)
    want = _run(q, k, v, parents, kc, vc, lengths, table)
    both = torch.stack((kc, vc), 2)                             # keys and values of a row side by side
    fused = torch.cat((q, k, v), 2)
    heads = torch.stack((kc, vc)).transpose(2, 3).contiguous().transpose(2, 3)      # heads before rows
    assert torch.equal(_run(fused[:, :, :4], fused[:, :, 4:6], fused[:, :, 6:], parents, both[:, :, 0], both[:, :, 1], lengths, table), want)
    assert torch.equal(_run(q, k, v, parents, heads[0], heads[1], lengths, table), want)
    odd = torch.zeros(*kc.shape[:3], 70, dtype=dtype, device=DEV)
    odd[..., 3:67] = kc
    x = (q, k, v, parents, odd[..., 3:67], vc, lengths, table)
    _check(_run(*x), *x, 0.125)


def test_offsets_beyond_32_bits():
    n = (1 << 31) // 128 + 100
    kc = torch.zeros(1, n, 1, 128, dtype=BF16, device=DEV)
    vc = torch.zeros_like(kc)
    g = torch.Generator().manual_seed(33)
    q, k, v = (torch.randn(1, 2, h, 128, generator=g).bfloat16().to(DEV) for h in (2, 1, 1))
    # one row near the end has nearly all of the weight
    kc[0, n - 3, 0] = 40 * q[0, 0, 0] / q[0, 0, 0].float().norm()
    vc[0, n - 3, 0] = 1
    out = sa.tree_attention(q, k, v, None, kc, vc, torch.tensor([n], dtype=torch.int32, device=DEV), scale=4.0)
    assert ((out[0, 0, 0] - 1).abs() < 2.0 ** -7).all()
    out = sa.tree_attention(q, k, v, None, kc, vc, torch.tensor([n - 3], dtype=torch.int32, device=DEV), scale=4.0)
    assert (out[0, 0, 0].abs() < 2.0 ** -7).any()


def test_other_stream_and_replayed_graph():
    q, k, v, parents, kc, vc, lengths, table = [t.to(DEV) for t in _case(4, 3, 8, 2, 128, 16, 64, BF16, 27)]
    lengths.fill_(900)
    want = sa.tree_attention(q, k, v, parents, kc, vc, lengths, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sa.tree_attention(q, k, v, parents, kc, vc, lengths, table)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = sa.tree_attention(q, k, v, parents, kc, vc, lengths, table)
    g = torch.Generator().manual_seed(28)
    for n in (0, 17, 1024):
        lengths.fill_(n)
        q.copy_(torch.randn(q.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        assert torch.equal(got, sa.tree_attention(q, k, v, parents, kc, vc, lengths, table))


def test_prompt_draft_accept_draft():
    """The operators together: prompts through rotary and causal attention into pages, a drafted tree over them, its accepted
    path into the pages, the next token; the last step is causal attention over the whole accepted text."""
    B, H, HK, D, page, width = 2, 8, 2, 128, 16, 8
    g = torch.Generator().manual_seed(41)
    f = sa.rotary_frequencies(D, device=DEV)
    make = lambda *s: torch.randn(*s, generator=g).bfloat16().to(DEV)
    lens = [37, 64]
    cu = torch.tensor([0, 37, 101], dtype=torch.int32, device=DEV)
    table = torch.randperm(B * width, generator=g).view(B, width).int().to(DEV)
    kc, vc = torch.full((2, B * width, page, HK, D), math.nan, dtype=BF16, device=DEV)
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    q, k, v = make(101, H, D), make(101, HK, D), make(101, HK, D)
    qr, kr = sa.rotary_embedding(q, k, f, cu_seqlens=cu)
    first = sa.causal_attention(qr, kr, v, cu)
    sa.cache_append(kr, v, kc, vc, lengths, table, cu_seqlens=cu)
    lengths += torch.tensor(lens, dtype=torch.int32, device=DEV)
    # drafts: node 2 follows 0, node 3 follows 2; 0 - 2 - 3 is accepted in the first sequence, 0 in the second
    parents = torch.tensor([[-1, 0, 0, 2], [-1, 0, -2, -2]], dtype=torch.int32, device=DEV)
    depth = torch.tensor([[0, 1, 1, 2], [0, 1, 0, 0]], dtype=torch.int32, device=DEV)
    q2, k2, v2 = make(B, 4, H, D), make(B, 4, HK, D), make(B, 4, HK, D)
    qr2, kr2 = sa.rotary_embedding(q2, k2, f, positions=lengths[:, None] + depth)
    drafted = sa.tree_attention(qr2, kr2, v2, parents, kc, vc, lengths, table)
    taken = torch.tensor([[0, 2, 3], [0, -1, -1]], dtype=torch.int32, device=DEV)
    sa.cache_append(kr2, v2, kc, vc, lengths, table, rows=taken)
    lengths += (taken >= 0).sum(1, dtype=torch.int32)
    q3, k3, v3 = make(B, 1, H, D), make(B, 1, HK, D), make(B, 1, HK, D)
    qr3, kr3 = sa.rotary_embedding(q3, k3, f, positions=lengths[:, None])
    last = sa.tree_attention(qr3, kr3, v3, None, kc, vc, lengths, table)
    for b in range(B):
        rows, path = slice(int(cu[b]), int(cu[b + 1])), [r for r in taken[b].tolist() if r >= 0]
        whole = [torch.cat((a[rows], c[b, path], d[b])) for a, c, d in ((qr, qr2, qr3), (kr, kr2, kr3), (v, v2, v3))]
        again = sa.causal_attention(*[t[None] for t in whole])[0]
        # both round softmax weights and result to bf16, in other orders: twice the bound of one, 2 * (2 * 2^-8) of the values'
        # weighted magnitude, which is below 1
        n = lens[b]
        for got, want in ((first[rows], again[:n]), (drafted[b, path], again[n:n + len(path)]), (last[b], again[-1:])):
            assert (got.double() - want.double()).abs().max() <= 4 * 2.0 ** -8

"""cache_append against indexing on the CPU: pages in any order, rows chosen from drafts, packed prompts, odd sizes, places
and pages outside of the cache, caches longer than 2^31 elements, capture into a graph."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _expect(k, v, kc, vc, lengths, table, page, rows=None, cu=None):
    """The definition, row by row, on CPU copies."""
    kc, vc = kc.cpu().clone(), vc.cpu().clone()
    k, v = k.cpu(), v.cpu()
    capacity = page * (table.shape[1] if table is not None else 1)
    for b, n in enumerate(lengths.tolist()):
        if cu is not None:
            taken = [(i, k[r], v[r]) for i, r in enumerate(range(cu[b], cu[b + 1]))]
        else:
            order = range(k.shape[1]) if rows is None else rows[b].tolist()
            taken = [(i, k[b, r], v[b, r]) for i, r in enumerate(order) if 0 <= r < k.shape[1]]
        for i, kr, vr in taken:
            place = n + i
            if n < 0 or place >= capacity:
                continue
            p = b if table is None else table[b, place // page].item()
            if 0 <= p < kc.shape[0]:
                kc[p, place % page], vc[p, place % page] = kr, vr
    return kc, vc


def _caches(shape, dtype, g):
    return [torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,N,HK,D,page,width", [
    (1, 1, 1, 1, 1, 3), (2, 1, 4, 128, 16, 4), (3, 5, 2, 64, 16, 2), (4, 33, 1, 80, 64, 3), (2, 7, 3, 33, 5, 6), (2, 300, 2, 64, 1000, 1)])
@pytest.mark.parametrize("paged", [True, False])
def test_rows_of_a_batch(B, N, HK, D, page, width, dtype, paged):
    g = torch.Generator().manual_seed(B + N + D)
    k, v = _caches((B, N, HK, D), dtype, g)
    pages = B * width + 2 if paged else B
    kc, vc = _caches((pages, page if paged else page * width, HK, D), dtype, g)
    capacity = page * width
    table = torch.randperm(pages, generator=g)[:B * width].view(B, width).int() if paged else None
    lengths = torch.randint(0, capacity + 1, (B,), generator=g).int()          # some run over the end
    lengths[0] = 0
    chosen = torch.randint(-1, N + 1, (B, 6), generator=g).int()
    place = page if paged else capacity
    on = lambda t: t.to(DEV) if t is not None else None
    for rows in (None, chosen):
        want = _expect(k, v, kc, vc, lengths, table, place, rows)
        sa.cache_append(k, v, kc, vc, lengths.to(DEV), on(table), rows=on(rows))
        assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (20, torch.float16), (128, torch.float32)])
def test_packed_rows_views_and_pages_that_are_none(D, dtype):
    g = torch.Generator().manual_seed(D)
    cu = [1, 1, 18, 19, 40]
    qkv = torch.randn(45, 7, D, generator=g).to(dtype).to(DEV)
    k, v = qkv[:, 3:5], qkv[:, 5:7]
    kc, vc = (t[:, :, 1:3] for t in _caches((6, 16, 4, D), dtype, g))            # heads of a larger cache
    table = torch.tensor([[5, 0], [3, 6], [-1, 1], [2, 4]]).int()                # 6 and -1: not the cache's
    lengths = torch.tensor([3, 9, 2, 14]).int()
    want = _expect(k, v, kc, vc, lengths, table, 16, cu=cu)
    sa.cache_append(k, v, kc, vc, lengths.to(DEV), table.to(DEV), cu_seqlens=torch.tensor(cu).int().to(DEV))
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


def test_offsets_beyond_32_bits():
    """A cache of 2^31 + elements: its last rows are reached, their mirror images 2^32 bytes before are not."""
    kc = torch.zeros(1, (1 << 31) // 128 + 64, 1, 128, dtype=torch.bfloat16, device=DEV)
    vc = torch.zeros_like(kc)
    k, v = (torch.full((1, 3, 1, 128), x, dtype=torch.bfloat16, device=DEV) for x in (1.0, 2.0))
    n = kc.shape[1] - 3
    sa.cache_append(k, v, kc, vc, torch.tensor([n], dtype=torch.int32, device=DEV))
    assert (kc[0, n:] == 1).all() and (vc[0, n:] == 2).all()
    assert kc[0, :n].count_nonzero() == 0 and vc[0, :n].count_nonzero() == 0


def test_replayed_graph():
    g = torch.Generator().manual_seed(9)
    k, v = _caches((2, 4, 2, 64), torch.bfloat16, g)
    kc, vc = _caches((4, 16, 2, 64), torch.bfloat16, g)
    table = torch.tensor([[3, 1], [0, 2]], dtype=torch.int32)
    lengths, rows = torch.tensor([0, 3], dtype=torch.int32, device=DEV), torch.tensor([[0, 2, -1], [1, 3, 3]], dtype=torch.int32, device=DEV)
    on = table.to(DEV)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        sa.cache_append(k, v, kc, vc, lengths, on, rows=rows)
    for _ in range(3):
        k.copy_(torch.randn(k.shape, generator=g))
        want = _expect(k, v, kc, vc, lengths.cpu(), table, 16, rows.cpu())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
        lengths += 3


def test_rows_that_are_the_caches_own():
    """Views of the cache as new rows, which the call's own places overlap: all are read first."""
    g = torch.Generator().manual_seed(29)
    kc, vc = (torch.randn(2, 600, 4, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    want = [c.clone() for c in (kc, vc)]
    for b, n in ((0, 7), (1, 200)):
        for w, c in zip(want, (kc, vc)):
            w[b, n:n + 400] = c[b, :400]
    sa.cache_append(kc[:, :400], vc[:, :400], kc, vc, torch.tensor([7, 200], dtype=torch.int32, device=DEV))
    assert torch.equal(kc, want[0]) and torch.equal(vc, want[1])

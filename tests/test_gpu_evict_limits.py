"""cache_evict at the longest cache that it takes, 2^31 - 65 rows: numbers of rows stay within 31 bits, sums of them do not."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS = (1 << 31) - 65


def _cache():
    bits = torch.empty(ROWS, dtype=torch.int16, device=DEV).random_()
    return bits, bits.clone().view(torch.float16).view(1, ROWS, 1, 1)


@pytest.mark.parametrize("keep,first,recent,heavy,dropped", [
    (ROWS - 1, 0, ROWS - 2, [1], [0]),                          # every row moves, by one place
    (ROWS - 3, ROWS - 8, 2, [ROWS - 8, ROWS - 5, ROWS - 3], [ROWS - 7, ROWS - 6, ROWS - 4])])
def test_the_longest_cache(keep, first, recent, heavy, dropped):
    (k_bits, k_cache), (v_bits, v_cache) = _cache(), _cache()
    weights = torch.zeros(1, 1, ROWS, device=DEV)
    weights[..., heavy] = 2.0
    kept, left = sa.cache_evict(k_cache, v_cache, weights, torch.tensor([ROWS], dtype=torch.int32, device=DEV), keep, first, recent)
    assert left[0, 0, keep:].count_nonzero() == 0
    for bits, cache in ((k_bits, k_cache), (v_bits, v_cache)):
        assert torch.equal(cache.view(torch.int16).flatten()[keep:], bits[keep:])
    at = 0
    for a, b in zip([0] + [x + 1 for x in dropped], dropped + [ROWS]):       # runs of rows that stay
        to = slice(at, at + b - a)
        at += b - a
        assert torch.equal(kept[0, 0, to], torch.arange(a, b, dtype=torch.int32, device=DEV)) and torch.equal(left[0, 0, to], weights[0, 0, a:b])
        for bits, cache in ((k_bits, k_cache), (v_bits, v_cache)):
            assert torch.equal(cache.view(torch.int16).flatten()[to], bits[a:b])
    assert at == keep


@pytest.mark.parametrize("B,HK", [(11, 6), (16, 8), (13, 10), (3, 2)])      # (66 and 128 heads: two workgroups share one, 130: none do, 6: four)
def test_heads_that_workgroups_share(B, HK):
    rows, keep, first, recent = 33_000, 8_300, 4, 4_000
    g = torch.Generator(device=DEV).manual_seed(B)
    k_cache, v_cache = (torch.randn(B, rows, HK, 8, generator=g, device=DEV).half() for _ in range(2))
    weights = torch.randint(0, 5000, (B, HK, rows), generator=g, device=DEV).float()     # (some are equal)
    lengths = torch.randint(keep, rows + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    lengths[0], lengths[1] = rows, 100
    old = k_cache.clone(), v_cache.clone()
    kept, left = sa.cache_evict(k_cache, v_cache, weights, lengths, keep, first, recent)
    place = torch.arange(rows, device=DEV)
    for b in range(B):
        n = int(lengths[b])
        if n <= keep:
            assert torch.equal(kept[b, :, :n], place[:n].int().expand(HK, n)) and (kept[b, :, n:] == -1).all() and torch.equal(left[b, :, :n], weights[b, :, :n])
            assert left[b, :, n:].count_nonzero() == 0 and torch.equal(k_cache[b], old[0][b]) and torch.equal(v_cache[b], old[1][b])
            continue
        rank = weights[b].masked_fill((place < first) | ((place >= n - recent) & (place < n)), float("inf")).masked_fill(place >= n, -1.0)
        want = rank.sort(dim=-1, descending=True, stable=True)[1][:, :keep].sort(-1)[0]
        assert torch.equal(kept[b].long(), want) and torch.equal(left[b, :, :keep], weights[b].gather(1, want)) and left[b, :, keep:].count_nonzero() == 0
        for cache, o in zip((k_cache, v_cache), old):
            assert torch.equal(cache[b, keep:], o[b, keep:])
            for h in range(HK):
                assert torch.equal(cache[b, :keep, h], o[b, want[h], h])

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

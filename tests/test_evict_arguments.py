"""Numbers and tensors that cache_evict refuses before anything reaches the GPU (no kernel is launched here)."""
import pytest
import torch

import simplical_attn_amd as sa


def _evict(k_cache, v_cache, keep=5, **kw):
    lengths, table = torch.tensor([3, 4], dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(2, 3)
    return sa.cache_evict(k_cache, v_cache, torch.zeros(2, k_cache.shape[2], 3 * k_cache.shape[1]), lengths, keep, page_table=table, **kw)


@pytest.mark.parametrize("first,recent", [(1 << 62, 1 << 62), ((1 << 63) - 1, 1), (1, (1 << 63) - 1), (1 << 32, 0), (0, 1 << 32), ((1 << 32) + 2, (1 << 63) - 1), (3, 3), (6, 0), (0, 6)])
def test_first_and_recent_rows_beyond_those_that_stay(first, recent):
    """Their sum passes 64 bits in some of these."""
    cache = torch.zeros(6, 16, 2, 8)
    with pytest.raises(ValueError, match="at most keep"):
        _evict(cache, cache.clone(), first=first, recent=recent)
    with pytest.raises(RuntimeError, match="GPU only"):
        _evict(cache, cache.clone(), first=3, recent=2)

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


def _halves():
    """Pairs of views of one buffer with no element in common."""
    a, b, c, d = torch.zeros(2, 6, 16, 2, 8), torch.zeros(6, 2, 16, 2, 8), torch.zeros(6, 16, 4, 8), torch.zeros(6, 16, 2, 20)
    e = torch.zeros(6 * 16 * 2 * 8 * 2)
    yield from ((a[0], a[1]), (b[:, 0], b[:, 1]), (b[:, 1], b[:, 0]), (c[:, :, :2], c[:, :, 2:]), (c[:, :, ::2], c[:, :, 1::2]), (d[..., :8], d[..., 12:]), (d[..., 8:16], d[..., :8]))
    yield e[:1536].view(6, 16, 2, 8), e[1536:].view(6, 16, 2, 8)
    yield b[:, 0], b.as_strided((6, 16, 2, 8), (512, 8, 128, 1), 256)       # (heads outside of rows there)


def _shared():
    """Pairs of views that share some elements."""
    a, c, d = torch.zeros(12, 16, 2, 8), torch.zeros(6, 32, 3, 8), torch.zeros(6, 16, 2, 24)
    yield from ((a[:6], a[:6]), (a[:6], a[5:11]), (a[3:9], a[:6]), (a[:6], a[1:7]), (a[::2], a[2::1][:6]), (c[:, :16, :2], c[:, 8:24, :2]), (c[:, :16, :2], c[:, :16, 1:]),
                (c[:, 16:, :2], c[:, 1:17, 1:]), (d[..., :8], d[..., 4:12]), (d[..., 7:15], d[..., :8]))
    flat = torch.zeros(2000)
    yield flat[:1536].view(6, 16, 2, 8), flat[1:1537].view(6, 16, 2, 8)
    yield a[:6], a.as_strided((6, 16, 2, 8), (512, 8, 128, 1), 256)


@pytest.mark.parametrize("pair", range(9))
def test_halves_of_one_buffer_are_two_caches(pair):
    k_cache, v_cache = list(_halves())[pair]
    with pytest.raises(RuntimeError, match="GPU only"):
        _evict(k_cache, v_cache)


@pytest.mark.parametrize("pair", range(12))
def test_caches_with_memory_in_common(pair):
    k_cache, v_cache = list(_shared())[pair]
    marks = [set(torch.arange(v.untyped_storage().nbytes() // 4).as_strided(v.shape, v.stride(), v.storage_offset()).flatten().tolist()) for v in (k_cache, v_cache)]
    assert marks[0] & marks[1]
    with pytest.raises(ValueError, match="same memory"):
        _evict(k_cache, v_cache)

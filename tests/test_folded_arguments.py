"""Tensors that are changed in place and whose own elements share memory are refused (no kernel is launched here)."""
import pytest
import torch

import simplical_attn_amd as sa

FLAT = torch.zeros(6000)


def _tree(weights):
    q, k, cache = torch.zeros(2, 1, 4, 8), torch.zeros(2, 1, 2, 8), torch.zeros(6, 16, 2, 8)
    lengths, table = torch.tensor([3, 4], dtype=torch.int32), torch.arange(6, dtype=torch.int32).view(2, 3)
    return sa.tree_attention(q, k, k, None, cache, cache, lengths, table, weights=weights)


def _sums(weights):
    return sa.key_weights(torch.zeros(2, 5, 4, 8), torch.zeros(2, 5, 2, 8), torch.zeros(2, 4, 5), weights=weights, lengths=torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("call", [_tree, _sums])
@pytest.mark.parametrize("strides,fine", [((96, 48, 1), True), ((48, 96, 1), True), ((200, 50, 1), True), ((40, 80, 1), False), ((96, 47, 1), False), ((48, 48, 1), False), ((1, 1, 1), False),
                                          ((95, 48, 1), False), ((1, 48, 1), False)])
def test_weights_that_are_added_to(call, strides, fine):
    weights = FLAT.as_strided((2, 2, 48), strides)
    distinct = torch.arange(6000).as_strided((2, 2, 48), strides).unique().numel() == weights.numel()
    assert distinct == fine
    with pytest.raises(RuntimeError if fine else ValueError, match="GPU only" if fine else "share memory"):
        call(weights)


@pytest.mark.parametrize("strides", [(256, 16, 8, 1), (512, 32, 16, 1), (16, 96, 8, 1), (256, 15, 8, 1), (256, 16, 7, 1), (255, 16, 8, 1), (256, 16, 16, 1), (8, 16, 8, 1), (128, 8, 800, 1)])
def test_caches(strides):
    k_cache, other = FLAT.as_strided((6, 16, 2, 8), strides), torch.zeros(6, 16, 2, 8)
    fine = torch.arange(6000).as_strided((6, 16, 2, 8), strides).unique().numel() == other.numel()
    for pair in ((k_cache, other), (other, k_cache)):
        with pytest.raises(RuntimeError if fine else ValueError, match="GPU only" if fine else "share memory"):
            sa.cache_evict(*pair, torch.zeros(2, 2, 48), torch.tensor([3, 4], dtype=torch.int32), 5, page_table=torch.arange(6, dtype=torch.int32).view(2, 3))

"""tree_attention with a window or gathered weights over long caches of several sequences: shares dealt by the sequences' lengths, and page
tables that do not fit a workgroup's LDS (more than 4096 pages in reach), against the definition in 64 bits."""
import pytest
import torch

from simplical_attn_amd import _lib
from tests.test_gpu_window_tree import BF16, DEV, FP16, FP32, _case, _check, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T,H,HK,D,page,width,dtype,flags", [
    (4, 1, 4, 2, 64, 64, 70, FP32, 0), (3, 1, 4, 1, 128, 16, 300, FP32, 0), (3, 5, 4, 2, 64, 64, 70, FP32, 0), (3, 1, 2, 1, 200, 64, 70, BF16, 0), (4, 3, 2, 2, 64, 64, 70, FP16, _lib.FLAG_FORCE_GENERIC),
    (3, 24, 4, 1, 128, 64, 80, BF16, 0), (4, 40, 4, 1, 64, 16, 300, FP16, 0), (3, 64, 4, 1, 128, 100, 50, FP16, 0)])
@pytest.mark.parametrize("window,sinks", [(2100, 5), (2500, 200), (4000, 0)])
def test_shares_dealt_by_length(B, T, H, HK, D, page, width, dtype, flags, window, sinks):
    """(from eight shares per sequence on: 1024 rows in reach, 2048 for large trees)"""
    q, k, v, parents, kc, vc, lengths, table = _case(B, T, H, HK, D, page, width, dtype, B + T + D)
    lengths[1], lengths[B - 1] = 0, 1234                    # (ragged: empty, and shorter than the window)
    before = torch.rand(B, HK, page * width, generator=torch.Generator().manual_seed(3)).to(DEV) if T == 1 else None
    after = None if before is None else before.clone()
    out = _run(q, k, v, parents, kc, vc, lengths, table, window, sinks, flags, weights=after)
    _check(out, q, k, v, parents, kc, vc, lengths, table, D ** -0.5, window, sinks, dtype != FP32 and not flags and D <= 128, before, after)


@pytest.mark.parametrize("B,D,dtype,flags", [(4, 64, FP32, 0), (3, 128, FP32, 0), (3, 96, BF16, _lib.FLAG_FORCE_GENERIC)])
def test_weights_over_dealt_shares(B, D, dtype, flags):
    q, k, v, _, kc, vc, lengths, table = _case(B, 1, 4, 2, D, 64, 70, dtype, B + D)
    lengths[1], lengths[2] = 0, 900
    before = torch.rand(B, 2, 64 * 70, generator=torch.Generator().manual_seed(3)).to(DEV)
    after = before.clone()
    out = _run(q, k, v, None, kc, vc, lengths, table, None, 0, flags, weights=after)
    _check(out, q, k, v, None, kc, vc, lengths, table, D ** -0.5, None, 0, False, before, after)


@pytest.mark.parametrize("T,H,D,dtype", [(1, 4, 128, BF16), (1, 4, 64, FP16), (1, 70, 64, BF16), (7, 2, 64, BF16), (20, 4, 128, FP16), (40, 4, 64, BF16)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (17000, 40), (30, 16500)])
def test_page_tables_that_do_not_fit(T, H, D, dtype, window, sinks):
    """5000 pages of four rows; some are none of the cache's."""
    if window is None and T > 1:
        pytest.skip("weights of single tokens, or a window, take these kernels")
    q, k, v, parents, kc, vc, lengths, table = _case(2, T, H, 1, D, 4, 5000, dtype, T + D)
    lengths[1] = 17311
    for bad in (False, True):
        if bad:
            table[0, ::7], table[0, 1], table[1, 2000:2100] = -1, 1 << 30, 10_003
        before = torch.rand(2, 1, 20_000, generator=torch.Generator().manual_seed(3)).to(DEV) if T == 1 else None
        after = None if before is None else before.clone()
        out = _run(q, k, v, parents, kc, vc, lengths, table, window, sinks, weights=after)
        _check(out, q, k, v, parents, kc, vc, lengths, table, D ** -0.5, window, sinks, True, before, after)

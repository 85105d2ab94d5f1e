"""key_weights of many packed sequences with many first keys: more shares of the first keys' blocks than are launched one by one."""
import pytest
import torch

import simplical_attn_amd as sa
from tests.test_gpu_key_weights import BF16, DEV, FP16, FP32, _check, _exact, _inputs, _lse

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,H,HK,D", [(BF16, 16, 8, 64), (FP16, 8, 8, 128), (FP32, 16, 8, 64)])
@pytest.mark.parametrize("sequences,rows,sinks", [(500, 80, 600), (3000, 40, 600)])
def test_blocks_of_first_keys_in_few_shares(sequences, rows, sinks, dtype, H, HK, D):
    """(65536 workgroups at most: shares of the whole stream in the first case, none in the second)"""
    window, g = 9, torch.Generator().manual_seed(sequences)
    lengths = torch.randint(0, rows, (sequences,), generator=g).tolist()
    lengths[5], lengths[100], lengths[-1] = 2100, 1, 700
    ends = [0]
    for n in lengths:
        ends.append(ends[-1] + n)
    q, k = _inputs((ends[-1] + 3,), H, HK, D, dtype, 7)
    cu = torch.tensor(ends, dtype=torch.int32, device=DEV)
    lse = _lse(q, k, cu, window, sinks)
    got = sa.key_weights(q, k, lse, cu, window=window, sinks=sinks)
    places, held = torch.zeros(sequences, HK, 2100, device=DEV), torch.zeros(sequences, dtype=torch.int32, device=DEV)
    sa.key_weights(q, k, lse, cu, window=window, sinks=sinks, weights=places, lengths=held)
    for i in [*range(8), *range(95, 105), sequences // 2, sequences - 1]:
        a, b = ends[i], ends[i + 1]
        for hk in (0, 3, HK - 1):
            hs = slice(hk * (H // HK), (hk + 1) * (H // HK))
            if b > a:
                _check(got[hk, a:b], _exact(q[a:b, hs], k[a:b, hk], lse[hs, a:b], D ** -0.5, window, sinks))
            assert torch.equal(places[i, hk, :b - a], got[hk, a:b]) and places[i, hk, b - a:].count_nonzero() == 0
    assert got[:, ends[-1]:].count_nonzero() == 0
    # every query's weights are one
    assert (got.double().sum(1) - ends[-1] * (H // HK)).abs().max() <= 1e-5 * ends[-1] * H

"""Windowed tree_attention over a cache whose one page has as many rows as a sequence may hold, 2^31 - 65."""
import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROWS, E = (1 << 31) - 65, 2.0 ** -24


@pytest.mark.parametrize("H,flags", [(2, 0), (80, 0), (2, _lib.FLAG_FORCE_GENERIC)])         # (80 rows: other kernels)
@pytest.mark.parametrize("T", [1, 2])
def test_one_page_of_all_rows(H, flags, T):
    D, window, sinks = 8, 100, 70
    g = torch.Generator(device=DEV).manual_seed(H + T)
    cache = torch.empty(1, ROWS, 1, D, dtype=torch.bfloat16, device=DEV)     # keys and values: it is only read
    cache[:, :200].normal_(generator=g)
    cache[:, -300:].normal_(generator=g)
    q, k, v = (torch.randn(1, T, h, D, generator=g, device=DEV).to(torch.bfloat16) for h in (H, 1, 1))
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    for held in (ROWS, ROWS - 77):
        lengths = torch.tensor([held], dtype=torch.int32, device=DEV)
        weights = torch.zeros(1, 1, ROWS, device=DEV) if T == 1 else None
        out = sa.tree_attention(q, k, v, None, cache, cache, lengths, table, None, flags, window, sinks, weights)
        for i in range(T):
            first, low = torch.arange(sinks), held + i - window + 1          # node i stands at place held + i
            rows = torch.cat((cache[0, :sinks, 0], cache[0, low:held, 0]))
            K, V = (torch.cat((rows, x[0, :i + 1, 0])).double() for x in (k, v))
            S = q[0, i].double() @ K.T * D ** -0.5
            P = torch.softmax(S, 1)
            want = P @ V
            r = (D + 4) * E * D ** -0.5 * (q[0, i].double().abs() @ K.abs().T).amax(1, keepdim=True)
            t = 2.0 ** -8                                                    # (bf16: half a step; of the weights where they are rounded, and of the result)
            rel = 2 * r + (len(K) + 16) * E
            assert ((out[0, i].double() - want).abs() <= (P @ V.abs()) * (rel + t) + t * want.abs() + 2.0 ** -133).all()
            if weights is not None:
                at = torch.cat((first, torch.arange(low, held))).to(DEV)
                sums, off = P.sum(0), (P * rel).sum(0) + (H + 2) * E * P.sum(0) + 2.0 ** -140
                assert ((weights[0, 0, at].double() - sums[:-1]).abs() <= off[:-1]).all()
                rest = sums[-1] if held < ROWS else 0.0                      # (the node's own has no place in a full cache)
                if held < ROWS:
                    assert (weights[0, 0, held].double() - rest).abs() <= off[-1]
                    weights[0, 0, held] = 0.0
                weights[0, 0, at] = 0.0
                assert weights.count_nonzero() == 0

"""Packed rows whose cu_seqlens reach beyond the rows: entries are taken as 0 or the number of rows, and nothing outside of the tensors
is read or written."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# (the smallest int: a row's number less that does not fit an int)
@pytest.mark.parametrize("first", [-2 ** 31, -2 ** 31 + 3, -5])
@pytest.mark.parametrize("last", [20, 2 ** 31 - 1])
def test_bounds_beyond_the_rows(first, last):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(20, h, 64, generator=g).to(DEV).bfloat16() for h in (4, 2, 2))
    inside, beyond = _ints(0, 7, 20), _ints(first, 7, last)
    f = sa.rotary_frequencies(64, device=DEV)
    for a, b in zip(sa.rotary_embedding(q, k, f, cu_seqlens=beyond), sa.rotary_embedding(q, k, f, cu_seqlens=inside)):
        assert torch.equal(a, b)
    caches = [[torch.zeros(6, 4, 2, 64, dtype=torch.bfloat16, device=DEV) for _ in range(2)] for _ in range(2)]
    table, lengths = _ints(0, 1, 2, 3, 4, 5).view(2, 3), _ints(2, 1)
    for cu, (kc, vc) in zip((beyond, inside), caches):
        sa.cache_append(k, v, kc, vc, lengths, table, cu_seqlens=cu)
    assert torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])
    dout = torch.randn(20, 4, 64, generator=g).to(DEV).bfloat16()
    for flags in (0, 1):
        results = []
        for cu in (beyond, inside):
            out, lse = sa.causal_attention_forward(q, k, v, cu, flags=flags)
            results.append((out, lse, *sa.causal_attention_backward(q, k, v, out, lse, dout, cu, flags=flags)))
        for a, b in zip(*results):
            assert torch.equal(a, b)

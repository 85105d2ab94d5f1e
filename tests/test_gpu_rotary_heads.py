"""rotary_embedding where q or k has no head."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_no_heads_of_one():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 9, 3, 64, generator=g).to(DEV)
    none, f = x[:, :, :0], sa.rotary_frequencies(64, device=DEV)
    want, _ = sa.rotary_embedding(x, None, f)
    a, b = sa.rotary_embedding(none, x, f)
    assert a.shape == none.shape and torch.equal(b, want)
    a, b = sa.rotary_embedding(x, none, f)
    assert b.shape == none.shape and torch.equal(a, want)
    leaf = x.clone().requires_grad_(True)
    _, b = sa.rotary_embedding(none, leaf, f)
    same = x.clone().requires_grad_(True)
    c, _ = sa.rotary_embedding(same, None, f)
    assert torch.equal(torch.autograd.grad(b, leaf, x)[0], torch.autograd.grad(c, same, x)[0])

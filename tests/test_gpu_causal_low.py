"""What rounding the output left, kept by causal_attention_forward and given to causal_attention_backward: the gradients are then those of
the training path."""
import pytest
import torch

import simplical_attn_amd as sa

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,D,flags", [(20, 64, 0), (300, 128, 0), (50, 136, 0), (90, 64, 1)])
def test_gradients_with_the_output_s_low_part(N, D, flags, dtype):
    g = torch.Generator().manual_seed(N)
    q, k, v, dout = (torch.randn(2, N, h, D, generator=g).to(dtype).to(DEV) for h in (4, 2, 2, 4))
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want = torch.autograd.grad(sa.causal_attention(*leaves, flags=flags), leaves, dout)
    out, lse, low = sa.causal_attention_forward(q, k, v, flags=flags, keep_low=True)
    plain = sa.causal_attention_forward(q, k, v, flags=flags)
    assert len(plain) == 2 and torch.equal(plain[0], out) and torch.equal(plain[1], lse)
    # half a step of the output, and itself rounded
    step = torch.finfo(dtype).eps / 2
    assert low.dtype == dtype and (low.double().abs() <= step * (1 + step) * out.double().abs() + 2.0 ** -25).all()
    for given in (low, low.transpose(1, 2).contiguous().transpose(1, 2)):          # (strides other than the output's)
        for a, b in zip(sa.causal_attention_backward(q, k, v, out, lse, dout, flags=flags, out_low=given), want):
            assert torch.equal(a, b)


def test_float32_has_none():
    q = torch.randn(1, 9, 2, 64, device=DEV)
    out, lse, low = sa.causal_attention_forward(q, q, q, keep_low=True)
    assert low is None and len(sa.causal_attention_backward(q, q, q, out, lse, q, out_low=low)) == 3


def test_empty():
    q = torch.zeros(1, 0, 2, 64, device=DEV, dtype=torch.float16)
    out, lse, low = sa.causal_attention_forward(q, q, q, keep_low=True)
    assert low.shape == q.shape and sa.causal_attention_backward(q, q, q, out, lse, q, out_low=low)[0].shape == q.shape

"""What causal_attention_backward refuses as out_low, before anything reaches the GPU."""
import pytest
import torch

import simplical_attn_amd as sa


@pytest.mark.parametrize("dtype,low", [
    (torch.float32, torch.zeros(1, 5, 4, 8)),
    (torch.float16, torch.zeros(1, 5, 2, 8, dtype=torch.float16)),
    (torch.float16, torch.zeros(1, 5, 4, 8, dtype=torch.bfloat16)),
])
def test_out_low(dtype, low):
    q = torch.zeros(1, 5, 4, 8, dtype=dtype)
    with pytest.raises(ValueError, match="out_low"):
        sa.causal_attention_backward(q, q, q, q, torch.zeros(1, 4, 5), q, out_low=low)

"""cache_append and inference tensors: refused outside of inference mode before anything is written, as every change in place is."""
import pytest
import torch

import simplical_attn_amd as sa


def _tensors(device, dtype=torch.bfloat16):
    with torch.inference_mode():
        kc, vc = (torch.zeros(2, 8, 1, 64, dtype=dtype, device=device) for _ in range(2))
    k = torch.ones(2, 3, 1, 64, dtype=dtype, device=device)
    return k, kc, vc, torch.zeros(2, dtype=torch.int32, device=device)


def test_refused():
    k, kc, vc, lengths = _tensors("cpu")
    for a, b in ((kc, vc), (kc.clone(), vc), (kc, vc.clone())):
        with pytest.raises(RuntimeError, match="inference mode"):
            sa.cache_append(k, k, a, b, lengths)


@pytest.mark.gpu
def test_nothing_is_written_outside_and_rows_are_inside():
    k, kc, vc, lengths = _tensors("cuda:0")
    with pytest.raises(RuntimeError, match="inference mode"):
        sa.cache_append(k, k, kc, vc, lengths)
    assert kc.count_nonzero() == 0 and vc.count_nonzero() == 0
    with torch.inference_mode():
        sa.cache_append(k, k, kc, vc, lengths)
    assert (kc[:, :3] == 1).all() and (vc[:, :3] == 1).all() and kc[:, 3:].count_nonzero() == 0

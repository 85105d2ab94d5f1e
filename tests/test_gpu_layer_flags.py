"""Kernels with fp32 products for 16-bit tensors, asked for by `flags`: in training and for drafted trees.  Bounds: causal_util.py, with
nothing rounded but the results."""
import math

import pytest
import torch

import simplical_attn_amd as sa
from simplical_attn_amd import _lib
from tests.causal_util import check, exact

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,H,HK,D", [(33, 2, 1, 64), (200, 4, 2, 128)])
def test_training_with_fp32_products(N, H, HK, D, dtype):
    g = torch.Generator().manual_seed(N)
    q, k, v, dout = (torch.randn(1, N, h, D, generator=g).to(dtype).to(DEV) for h in (H, HK, HK, H))
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = sa.causal_attention(*leaves, flags=_lib.FLAG_FORCE_GENERIC)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    G = H // HK
    for hk in range(HK):
        hs = slice(hk * G, hk * G + G)
        want = exact(q[0, :, hs].detach(), k[0, :, hk].detach(), v[0, :, hk].detach(), dout[0, :, hs], D ** -0.5, dtype, False)
        for name, x in (("out", out[0, :, hs]), ("dq", dq[0, :, hs]), ("dk", dk[0, :, hk:hk + 1]), ("dv", dv[0, :, hk:hk + 1])):
            check(x, want[name], name)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,H,D", [(1, 4, 128), (20, 4, 64)])
def test_trees_with_fp32_products(T, H, D, dtype):
    n, E = 500, 2.0 ** -24
    g = torch.Generator().manual_seed(T)
    q, k, v, kc, vc = (torch.randn(1, m, h, D, generator=g).to(dtype).to(DEV) for m, h in ((T, H), (T, 1), (T, 1), (n, 1), (n, 1)))
    out = sa.tree_attention(q, k, v, None, kc, vc, torch.tensor([n], dtype=torch.int32, device=DEV), flags=_lib.FLAG_FORCE_GENERIC)
    K, V = (torch.cat((c[0, :, 0], x[0, :, 0])).double() for c, x in ((kc, k), (vc, v)))
    seen = torch.arange(n + T, device=DEV)[None] <= n + torch.arange(T, device=DEV)[:, None]
    for h in range(H):
        Q = q[0, :, h].double()
        P = torch.softmax((Q @ K.T * D ** -0.5).masked_fill(~seen, -math.inf), 1)
        r = ((D + 4) * E * D ** -0.5 * (Q.abs() @ K.abs().T)).amax(1, keepdim=True)
        want = P @ V
        # scores off by r, weights not rounded, sums of n + T terms, the result's own rounding
        bound = (P @ V.abs()) * (2 * r + (n + T + 16) * E) + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
        assert ((out[0, :, h].double() - want).abs() <= bound).all()

"""Causal attention of one sequence and one head in 64 bits, with bounds on how far a kernel's results may be off.

The bounds follow the arithmetic step by step (e = 2^-24, half a step of fp32; t: half a step of the tensors' type; w: half a
step of what softmax weights and dS are rounded to before they are multiplied on, t in the 16-bit kernels, e in the others):
  scores    s_ij off by r_i = max_j (D + 4) e scale sum_d |q||k|
  weights   relative to their sum: 2 r_i + w + (n + 16) e, n keys; out adds its own rounding; fp16 weights below its
            smallest normal number are off by 2^-25 of the largest one
  lse       r_i + (n + 16) e + 2 e |lse|
  dP        (D + 4) e sum |dO||v|; delta is formed from the rounded output: sum |dO| (error of out) + (D + 4) e sum |dO||out|
  dS        P (errors of dP and delta) + |dS| (error of P, from s and lse) + |dS| w
and the gradients sum those errors over their rows or columns, plus (n + 16) e of the magnitudes and their own rounding."""
import math

import torch

E = 2.0 ** -24


def exact(q, k, v, dout, scale, dtype, rounded):
    """q, dout [n, G, D] of the G heads that share k, v [n, D]; returns {name: (value, bound)}, heads joined as they are."""
    n, G, D = q.shape
    t = torch.finfo(dtype).eps / 2
    w = t if rounded else E
    low = 2.0 ** -25 if rounded and dtype == torch.float16 else 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    K, V = k.double(), v.double()
    mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    res = {name: [] for name in ("out", "lse", "dq")}
    dk, dv, bk, bv = torch.zeros_like(K), torch.zeros_like(V), torch.zeros_like(K), torch.zeros_like(V)
    for g in range(G):
        Q, dO = q[:, g].double(), dout[:, g].double()
        S = (Q @ K.T * scale).masked_fill(~mask, -math.inf)
        r = ((D + 4) * E * abs(scale) * (Q.abs() @ K.abs().T)).masked_fill(~mask, 0).amax(1, keepdim=True)
        P = torch.softmax(S, 1)
        out, lse = P @ V, torch.logsumexp(S, 1)
        rel = 2 * r + w + (n + 16) * E
        b_out = (P @ V.abs()) * rel + low * (mask.double() @ V.abs()) + t * out.abs() + tiny
        b_lse = r[:, 0] + (n + 16) * E + 2 * E * lse.abs()
        dP = dO @ V.T
        delta = (dO * out).sum(1, keepdim=True)
        b_dP = (D + 4) * E * (dO.abs() @ V.abs().T)
        b_delta = (dO.abs() * b_out).sum(1, keepdim=True) + (D + 4) * E * (dO * out).abs().sum(1, keepdim=True)
        rel_P = 2 * r + 2 * b_lse[:, None] + 16 * E
        dS = P * (dP - delta)
        dS[0] = 0
        b_dS = (P * (b_dP + b_delta) + dS.abs() * (rel_P + w)) + low * mask
        dq = scale * (dS @ K)
        b_dq = abs(scale) * (b_dS @ K.abs() + (n + 16) * E * (dS.abs() @ K.abs()))
        res["out"].append((out, b_out))
        res["lse"].append((lse, b_lse))
        res["dq"].append((dq, b_dq + t * (dq.abs() + b_dq) + tiny))
        dk += scale * (dS.T @ Q)
        bk += abs(scale) * (b_dS.T @ Q.abs() + (n * G + 16) * E * (dS.abs().T @ Q.abs()))
        dv += P.T @ dO
        bv += ((rel_P + w) * P + low * mask).T @ dO.abs() + (n * G + 16) * E * (P.T @ dO.abs())
    both = {name: tuple(torch.stack(x, 1) for x in zip(*pairs)) for name, pairs in res.items()}
    both["dk"] = (dk[:, None], (bk + t * (dk.abs() + bk) + tiny)[:, None])
    both["dv"] = (dv[:, None], (bv + t * (dv.abs() + bv) + tiny)[:, None])
    return both


def check(got, bounds, what):
    want, bound = bounds
    x = got.double()
    assert torch.isfinite(x).all(), what
    far = (x - want).abs() / bound
    assert far.max() <= 1, "%s: %.3g of its bound off" % (what, far.max().item())

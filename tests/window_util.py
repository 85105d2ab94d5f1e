"""Windowed attention of one sequence in 64 bits, with bounds on how far a kernel's results may be off: those of causal_util.py
(e, t, w as there), summed over the keys that a query sees, n the most of them."""
import math

import torch

from tests.causal_util import E


def sees(n, window, sinks, device="cpu"):
    """[n, n]: whether query i sees key j."""
    i = torch.arange(n, device=device)
    i, j = i[:, None], i[None]
    return (j <= i) & ((i - j < window) | (j < sinks))


def exact(q, k, v, dout, scale, dtype, rounded, window, sinks):
    """q, dout [n, G, D] of the G heads that share k, v [n, D]; returns {name: (value, bound)}, heads joined as they are."""
    rows, G, D = q.shape
    t = torch.finfo(dtype).eps / 2
    w = t if rounded else E
    low = 2.0 ** -25 if rounded and dtype == torch.float16 else 0.0
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    K, V = k.double(), v.double()
    mask = sees(rows, window, sinks, q.device)
    n = int(mask.sum(1).max())
    alone = mask.sum(1) == 1                       # one weight, 1, whose gradient is zero
    most = int(mask.sum(0).max()) * G              # terms of a key's gradient
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
        dS[alone] = 0
        b_dS = (P * (b_dP + b_delta) + dS.abs() * (rel_P + w)) + low * mask
        dq = scale * (dS @ K)
        b_dq = abs(scale) * (b_dS @ K.abs() + (n + 16) * E * (dS.abs() @ K.abs()))
        res["out"].append((out, b_out))
        res["lse"].append((lse, b_lse))
        res["dq"].append((dq, b_dq + t * (dq.abs() + b_dq) + tiny))
        dk += scale * (dS.T @ Q)
        bk += abs(scale) * (b_dS.T @ Q.abs() + (most + 16) * E * (dS.abs().T @ Q.abs()))
        dv += P.T @ dO
        bv += ((rel_P + w) * P + low * mask).T @ dO.abs() + (most + 16) * E * (P.T @ dO.abs())
    both = {name: tuple(torch.stack(x, 1) for x in zip(*pairs)) for name, pairs in res.items()}
    both["dk"] = (dk[:, None], (bk + t * (dk.abs() + bk) + tiny)[:, None])
    both["dv"] = (dv[:, None], (bv + t * (dv.abs() + bv) + tiny)[:, None])
    return both

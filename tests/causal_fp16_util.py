"""Causal attention in 64 bits for fp16 tensors, with bounds on what values below fp16's smallest normal number may cost.

Beside the roundings that causal_util.py counts (scores r, weights and dS half a step w, sums (n + 16) e), a number below 2^-14 is off
by up to 2^-25 when it is rounded to fp16.  The kernels multiply what they round by powers of two first:
  out   weights by 2^L, L = log2(n) - 14, rounded up, from 0 to 8, over a reference point no higher than the row's maximum: off by
        2^-(25 + L) of the largest weight
  dv    weights by 2^15: 2^-40
  dq    dS of row i so that a bound of it, b_i = |dO_i| max_j |v_j| + |delta_i| over the keys that it sees, becomes 2^13 to 2^14: 2^-38 b_i
  dk    dS of key j the same with b_j = max_i |dO_i| |v_j| + max_i |delta_i| over the rows that see it, of all heads: 2^-38 b_j
(|.| of rows: Euclidean norms.)  dS in two parts is off by less than dS in one."""
import math

import torch

E, T = 2.0 ** -24, 2.0 ** -11
TINY = 2.0 ** -24


def exact(q, k, v, dout, scale):
    """q, dout [n, G, D] of the G heads that share k, v [n, D]; returns {name: (value, bound)}: out, dq [n, G, D], dk, dv [n, D]."""
    n, G, D = q.shape
    Q, K, V, dO = q.double(), k.double(), v.double(), dout.double()
    mask = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    norm_v = V.norm(dim=-1)
    seen_v = norm_v.cummax(0).values
    low_out = 2.0 ** (-25 - ((torch.arange(n, device=q.device) + 1.0).log2().ceil() - 14).clamp(0, 8)).double()[:, None]
    res = {"out": [], "dq": []}
    rows, dk, dv, bk, bv = [], torch.zeros_like(K), torch.zeros_like(V), torch.zeros_like(K), torch.zeros_like(V)
    for g in range(G):
        S = (Q[:, g] @ K.T * scale).masked_fill(~mask, -math.inf)
        r = ((D + 4) * E * abs(scale) * (Q[:, g].abs() @ K.abs().T)).masked_fill(~mask, 0).amax(1, keepdim=True)
        P = torch.softmax(S, 1)
        out, lse = P @ V, torch.logsumexp(S, 1)
        b_out = (P @ V.abs()) * (2 * r + T + (n + 16) * E) + low_out * (mask.double() @ V.abs())
        b_lse = r[:, 0] + (n + 16) * E + 2 * E * lse.abs()
        res["out"].append((out, b_out + T * out.abs() + TINY))
        dP = dO[:, g] @ V.T
        delta = (dO[:, g] * out).sum(1, keepdim=True)
        b_dP = (D + 4) * E * (dO[:, g].abs() @ V.abs().T)
        # (the output with what its rounding left: 2^-22 of it, or 2^-25 of the smallest normal number)
        b_delta = (dO[:, g].abs() * (b_out + 2.0 ** -22 * out.abs() + TINY)).sum(1, keepdim=True) + (D + 4) * E * (dO[:, g] * out).abs().sum(1, keepdim=True)
        rel_P = 2 * r + 2 * b_lse[:, None] + 16 * E
        dS = P * (dP - delta)
        dS[0] = 0
        rows.append((P, dS, P * (b_dP + b_delta) + dS.abs() * (rel_P + T), rel_P, dO[:, g].norm(dim=-1), delta[:, 0].abs()))
    last = lambda x: torch.stack(x).amax(0).flip(0).cummax(0).values.flip(0)      # over the rows from this one on, of all heads
    reach = last([x[4] for x in rows]) * norm_v + last([x[5] for x in rows])
    for g, (P, dS, b_dS, rel_P, norm, delta) in enumerate(rows):
        dq = scale * (dS @ K)
        b = b_dS + 2.0 ** -38 * (norm * seen_v + delta)[:, None] * mask
        b_dq = abs(scale) * (b @ K.abs() + (n + 16) * E * (dS.abs() @ K.abs()))
        res["dq"].append((dq, b_dq + T * (dq.abs() + b_dq) + TINY))
        b = b_dS + 2.0 ** -38 * reach[None] * mask
        dk += scale * (dS.T @ Q[:, g])
        bk += abs(scale) * (b.T @ Q[:, g].abs() + (n * G + 16) * E * (dS.abs().T @ Q[:, g].abs()))
        dv += P.T @ dO[:, g]
        bv += ((rel_P + T) * P + 2.0 ** -40 * mask).T @ dO[:, g].abs() + (n * G + 16) * E * (P.T @ dO[:, g].abs())
    both = {name: tuple(torch.stack(x, 1) for x in zip(*pairs)) for name, pairs in res.items()}
    both["dk"] = (dk, bk + T * (dk.abs() + bk) + TINY)
    both["dv"] = (dv, bv + T * (dv.abs() + bv) + TINY)
    return both

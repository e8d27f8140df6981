"""Oracle of attention within packed sequences: TEST INFRASTRUCTURE, not product code.

The formula in 64 bits, sequence by sequence and head by head, its gradients, and for each result how far it may lie from that when it is formed as the kernels say:
scores, exponentials and sums in fp32, probabilities and the scores' gradients rounded to the inputs' type where they multiply values, keys and queries, results rounded once.
Worst cases, added up: delta is allowed the output's whole bound, though the kernels form it of the output and of what rounding left of it, and dQ one rounding of the scores' gradients, which multiply
keys as two values.  How much nearer these bring the gradients is held by norms (tests/test_gpu_packed_gradients.py).
"""
from __future__ import annotations

import math

import torch


def packed(q, k, v, offsets, key_offsets, causal, scale, dout=None):
    """([o, dq, dk, dv], [their bounds]) in 64 bits (o alone without dout).  offsets: lists of whole numbers."""
    dt = q.dtype
    half = torch.finfo(dt).eps / 2                 # of one rounding to the inputs' type
    f = 2.0 ** -24                                 # of one in fp32
    # what is rounded to the type loses half of its smallest step; exponentials below 2^-126 are zero, and so may be operands of products that are (a probability 2^-126 off
    # is a term of a sum 2^-126 off, times what it multiplies)
    step = max(torch.finfo(dt).tiny * torch.finfo(dt).eps / 2, 2.0 ** -126)
    (_, H, D), Hk = q.shape, k.shape[1]
    outs = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, q, k, v)]
    bounds = [torch.zeros_like(t) for t in outs]
    for s in range(len(offsets) - 1):
        rows, keys = slice(offsets[s], offsets[s + 1]), slice(key_offsets[s], key_offsets[s + 1])
        Lq, Lk = offsets[s + 1] - offsets[s], key_offsets[s + 1] - key_offsets[s]
        if Lq <= 0 or Lk <= 0:
            continue
        at = torch.arange(Lk, device=q.device)[None, :] - Lk, torch.arange(Lq, device=q.device)[:, None] - Lq
        seen = at[0] <= at[1] if causal else torch.ones((Lq, Lk), dtype=torch.bool, device=q.device)
        for h in range(H):
            hk = h // (H // Hk)
            Q, K, V = q[rows, h].double(), k[keys, hk].double(), v[keys, hk].double()
            score = scale * (Q @ K.T)
            score = torch.where(seen, score, -math.inf)
            top = score.amax(-1, keepdim=True)
            top = torch.where(torch.isinf(top), 0.0, top)
            e = torch.exp(score - top)
            total = e.sum(-1, keepdim=True)
            P = torch.where(total > 0, e / torch.where(total > 0, total, 1.0), 0.0)
            # a score's error relative to 1 (its exponential's relative one): D products and sums, the scale, the difference to the maximum, the exponential
            off = f * (scale * (D + 4) * (Q.abs() @ K.abs().T) + 2 * top.abs() + 8)
            off = torch.where(seen, off, 0.0)
            off = off + off.amax(-1, keepdim=True) + (Lk + 16) * f       # and the sum's, by which it is divided
            o = P @ V
            outs[0][rows, h] = o
            # the probability and the output rounded, and the sum of rounded probabilities that it is divided by
            bounds[0][rows, h] = (P * (2 * half + 2 * off) + 2 * step) @ V.abs() + half * o.abs() + step
            if dout is None:
                continue
            dO = dout[rows, h].double()
            dP = dO @ V.T
            delta = (dO * o).sum(-1, keepdim=True)
            dS = P * (dP - delta) * scale
            outs[1][rows, h] = dS @ K
            outs[2][keys, hk] += dS.T @ Q
            outs[3][keys, hk] += P.T @ dO
            absolute = (D + 4) * f * (dO.abs() @ V.abs().T) + (D + 4) * f * (dO.abs() * o.abs()).sum(-1, keepdim=True) + (dO.abs() * bounds[0][rows, h]).sum(-1, keepdim=True)
            of_ds = dS.abs() * (half + off + 4 * f) + P * scale * absolute * 1.001 + step * (2 + (dP - delta).abs() * scale)
            sums = (Lk + H * Lq + 16) * f
            bounds[1][rows, h] = (of_ds + sums * dS.abs()) @ K.abs() + half * (dS @ K).abs()
            bounds[2][keys, hk] += (of_ds + sums * dS.abs()).T @ Q.abs()
            bounds[3][keys, hk] += (P * (half + off + sums) + step).T @ dO.abs()
    for i in (2, 3):
        bounds[i] += half * outs[i].abs()
    for b in bounds:
        b += step
    n = 1 if dout is None else 4
    return outs[:n], bounds[:n]

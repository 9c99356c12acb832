"""CPU oracle of attention over packed sequences and over a paged key-value cache, from the definitions in 64 bits (test infrastructure; never imported by the package).

Beside each value stands a bound on how far 16-bit kernels with fp32 sums may be from it, element for element, from counting roundings:
  * u = eps / 2 of the 16-bit type: one for P (or dS) as the operand of a product, one for the result.  fp16 has subnormals below 2^-14: an absolute 2^-25 for each operand
    besides (weights relative to a row's largest, which is 1 at least).
  * scores: D products added in fp32, off by D 2^-24 sum |q k| c at most; exp and its argument 4 2^-24 (1 + |s|); both enter numerator and denominator.
  * sums of n terms in fp32: n 2^-24 of the sum of their magnitudes.
"""
from __future__ import annotations

import math

import torch

F32 = 2.0 ** -24


def _u(dtype):
    return torch.finfo(dtype).eps / 2, (2.0 ** -25 if dtype == torch.float16 else 0.0)


def visible(lq, lk, causal):
    t, j = torch.arange(lq)[:, None], torch.arange(lk)[None]
    return (j <= t + lk - lq) if causal else torch.ones(lq, lk, dtype=torch.bool)


def attend(q, k, v, mask, scale):
    """One head of one sequence in 64 bits: (o, lse, P, s, relative error of P in fp32)."""
    s = q @ k.t() * scale
    s = torch.where(mask, s, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    P = torch.where(mask, torch.exp(s - torch.where(lse.isinf(), torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(s))
    size = torch.where(mask, (q.abs() @ k.abs().t()) * abs(scale), torch.zeros_like(s))
    top = size.amax(-1, keepdim=True) if k.shape[0] else torch.zeros(q.shape[0], 1, dtype=torch.float64)
    off = 2 * F32 * ((q.shape[1] + 4) * top + 8 + k.shape[0])
    return P @ v, lse, P, s, off


def ragged_fwd(q, k, v, cu_q, cu_k, causal, scale, dtype, rest=False):
    """(o, lse, bound of o, bound of lse); rows of no sequence: zeros, -inf.  `rest`: o as the sum of its rounding and what that left off, rounded too."""
    q, k, v = (x.double().cpu() for x in (q, k, v))
    Tq, Hq, D = q.shape
    group = Hq // k.shape[1]
    o, lse = torch.zeros_like(q), torch.full((Hq, Tq), -math.inf, dtype=torch.float64)
    o_tol, lse_tol = torch.zeros_like(q), torch.zeros_like(lse)
    u, tiny = _u(dtype)
    for a, b, c, d in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        mask = visible(b - a, d - c, causal)
        for h in range(Hq):
            K, V = k[c:d, h // group], v[c:d, h // group]
            o[a:b, h], lse[h, a:b], P, _, off = attend(q[a:b, h], K, V, mask, scale)
            size = P @ V.abs()
            o_tol[a:b, h] = (u + off) * size + (u * u if rest else u) * o[a:b, h].abs() + tiny * (V.abs().sum(0) + 2)
            lse_tol[h, a:b] = off[:, 0] + 8 * F32 * lse[h, a:b].abs().nan_to_num(posinf=0)
    return o, lse, o_tol, lse_tol


def ragged_bwd(q, k, v, dout, cu_q, cu_k, causal, scale, dtype, rest=False):
    """((dq, dk, dv), (their bounds)) of the forward's o, whose 16-bit rounding the row sums do . o have (`rest`: that of its rounding and the rest)."""
    q, k, v, g = (x.double().cpu() for x in (q, k, v, dout))
    Hq, D = q.shape[1:]
    group = Hq // k.shape[1]
    grads, tols = [torch.zeros_like(x) for x in (q, k, v)], [torch.zeros_like(x) for x in (q, k, v)]
    u, tiny = _u(dtype)
    o_tol = ragged_fwd(q, k, v, cu_q, cu_k, causal, scale, dtype, rest)[2]
    for a, b, c, d in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        mask = visible(b - a, d - c, causal)
        for h in range(Hq):
            Q, G, K, V = q[a:b, h], g[a:b, h], k[c:d, h // group], v[c:d, h // group]
            o, lse, P, s, off = attend(Q, K, V, mask, scale)
            off = off + 8 * F32 * lse.abs().nan_to_num(posinf=0)[:, None]
            dP, size = G @ V.t(), G.abs() @ V.abs().t()
            delta, delta_tol = (G * o).sum(-1, keepdim=True), (G.abs() * (o_tol[a:b, h] + (D + 2) * F32 * o.abs())).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            far = P * (delta_tol + (D + 2) * F32 * size + off * (dP.abs() + delta.abs())) + u * dS.abs() + tiny * mask
            sums = F32 * (b - a) * group
            grads[0][a:b, h] = scale * dS @ K
            tols[0][a:b, h] = abs(scale) * (far + (d - c) * F32 * dS.abs()) @ K.abs()
            grads[1][c:d, h // group] += scale * dS.t() @ Q
            tols[1][c:d, h // group] += abs(scale) * (far + sums * dS.abs()).t() @ Q.abs()
            grads[2][c:d, h // group] += P.t() @ G
            tols[2][c:d, h // group] += ((u + off + sums) * P + tiny * mask).t() @ G.abs()
    # (the result's own rounding, once, and that of the few intermediate steps in fp32)
    return grads, [t * (1 + u) + (u + 4 * F32) * x.abs() + 2 * tiny for t, x in zip(tols, grads)]


# ---- a paged cache, held as a list of lists of rows: what it stands for, not how it lies
def quantise(x, kind):
    """(codes, scale) of rows [..., D] as the definition has them, in fp32."""
    x = x.float()
    top = x.abs().amax(-1)
    by = torch.tensor(1 / 448 if kind == torch.float8_e4m3fn else 1 / 127, dtype=torch.float32)
    scale = torch.where(x.isfinite().all(-1), top * by, torch.full_like(top, math.nan))
    some = scale > 0
    y = torch.where(some[..., None], x / torch.where(some, scale, torch.ones_like(scale))[..., None], torch.zeros_like(x))
    return (y.round() if kind == torch.int8 else y).to(kind), scale


def dequantise(codes, scale):
    return codes.float().double() * scale.double()[..., None]


def decode(q, keys, values, scale, dtype):
    """One token of each sequence over its rows (lists of [n, Hkv, D] in 64 bits): (o, lse, their bounds)."""
    q = q.double().cpu()
    B, Hq, D = q.shape
    o, lse = torch.zeros_like(q), torch.full((B, Hq), -math.inf, dtype=torch.float64)
    o_tol, lse_tol = torch.zeros_like(q), torch.zeros_like(lse)
    for i, (k, v) in enumerate(zip(keys, values)):
        n = k.shape[0]
        if not n:
            continue
        O, L, OT, LT = ragged_fwd(q[i:i + 1], k, v, [0, 1], [0, n], False, scale, dtype)
        # (weights in fp16 are relative to the largest scale of a row of V as well: their subnormals are worth up to the largest element)
        o[i], lse[i], lse_tol[i] = O[0], L[:, 0], LT[:, 0]
        o_tol[i] = OT[0] + (2.0 ** -25 * n * v.abs().max() if dtype == torch.float16 else 0.0) + 4 * F32 * o[i].abs()
    return o, lse, o_tol, lse_tol

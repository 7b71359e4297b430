"""Attention and rotary positions by their formulas in 64 bits (CPU), with bounds on what rounding may do to a kernel's results.

Test infrastructure only."""
from __future__ import annotations

import math

import torch


def visible(B, S, T, causal, lengths, starts):
    """[B, S, T]: whether query i of sequence b sees key j."""
    key = torch.arange(T)
    held = torch.full((B,), T) if lengths is None else lengths.long().clamp(0, T)
    at = torch.arange(S) + (torch.full((B, 1), T - S) if starts is None else starts.long()[:, None])
    seen = (key < held[:, None])[:, None].expand(B, S, T)
    return seen & (key <= at[..., None]) if causal else seen


def attention(q, k, v, go=None, causal=True, scale=None, lengths=None, starts=None, exact_scores=False):
    """(out, dq, dk, dv, bounds): results in fp64 and, for tensors of q's type, how far each element may be off.

    With u half a step of the type (0 inside fp32 kernels, whose probabilities are not rounded again) and e = 2^-24:
    a score is off by (d + 8) e sum|q k|, so a probability by that, twice (numerator and sum), and by the few roundings of
    exponent and logarithm relative to itself; sums over n terms by n e of the sum of their absolute values; probabilities and
    score gradients are rounded to the type before the second product, results at the end; the backward pass reads the
    rounded output.  The hardware's 2^x gives 0 for what is below the normal numbers, so that a probability is off by
    2^-126 in absolute terms too, and what is made of it by that times what multiplies it.

    exact_scores: q k, and its distance from a row's largest, are numbers that fp32 holds.  A probability is then off by the
    rounding of that distance x times the scale times log2(e), twice (the factor's own and the product's), and by the 16 e of
    exponent and logarithm; the row's sum by what its terms are off on average."""
    B, S, H, d = q.shape
    T, G = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * u           # half a step of the subnormal numbers
    inner = 0.0 if q.dtype == torch.float32 else u
    e = 2.0 ** -24
    Q = q.double().transpose(1, 2)
    seen = visible(B, S, T, causal, lengths, starts)[:, None]
    held = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T) < lengths.long()[:, None]
    K, V = (torch.where(held[:, :, None, None], t.double(), 0.0).transpose(1, 2).repeat_interleave(H // G, 1) for t in (k, v))
    s = Q @ K.transpose(2, 3) * scale
    top = s.masked_fill(~seen, -math.inf).amax(-1, keepdim=True) if T else torch.full((B, H, S, 1), -math.inf)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.where(seen, (s - top).exp(), 0.0)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ V
    size = (Q.abs() @ K.abs().transpose(2, 3) * scale).masked_fill(~seen, 0.0)
    off = size.amax(-1, keepdim=True) if T else torch.zeros(B, H, S, 1)
    ep = 2 * ((d + 8) * e * off + 16 * e + 4 * e * top.abs())            # relative, of a probability
    if exact_scores:
        ep = 2 * e * torch.where(seen, top - s, 0.0) + 16 * e
        ep = ep + (p * ep).sum(-1, keepdim=True)
    lost = 2.0 ** -126 * seen.double()
    b_out = (p * (ep + T * e + inner)) @ V.abs() + lost @ V.abs() + u * out.abs() + tiny

    def last(x):
        return x.transpose(1, 2)
    if go is None:
        return (last(out),), (last(b_out),)
    g = go.double().transpose(1, 2)
    dv = p.transpose(2, 3) @ g
    dp = g @ V.transpose(2, 3)
    delta = (g * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    b_delta = (g.abs() * (b_out + d * e * out.abs())).sum(-1, keepdim=True)
    b_ds = p * (d * e * (g.abs() @ V.abs().transpose(2, 3)) + b_delta + 2 * e * (dp.abs() + delta.abs())) + (ep + inner) * ds.abs()
    b_ds = b_ds + lost * (dp.abs() + delta.abs())
    dq = ds @ K * scale
    b_dq = (b_ds + T * e * ds.abs()) @ K.abs() * scale + u * dq.abs() + tiny
    n = S * (H // G)
    dk = ds.transpose(2, 3) @ Q * scale
    b_dk = (b_ds + n * e * ds.abs()).transpose(2, 3) @ Q.abs() * scale
    b_dv = (p * (ep + inner + n * e) + lost).transpose(2, 3) @ g.abs()
    dk, dv, b_dk, b_dv = (x.reshape(B, G, H // G, T, d).sum(2) for x in (dk, dv, b_dk, b_dv))
    b_dk, b_dv = b_dk + u * dk.abs() + tiny, b_dv + u * dv.abs() + tiny
    return tuple(map(last, (out, dq, dk, dv))), tuple(map(last, (b_out, b_dq, b_dk, b_dv)))


def rotary(x, theta, positions, interleaved=False, size=1.0, inverse=False):
    """(result, bound): x [B, S, heads, d] with its first 2 * len(theta) elements turned, positions [B, S]."""
    R = 2 * len(theta)
    angle = positions.double()[:, :, None, None] * torch.tensor(theta, dtype=torch.float64)
    cos, sin = size * angle.cos(), size * angle.sin() * (-1 if inverse else 1)
    y = x.double().clone()
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    xa, xb = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = xa * cos - xb * sin, xb * cos + xa * sin
    # sine, cosine, their factor, two products and a sum in fp32: 6 roundings of numbers no larger than size * (|a| + |b|);
    # the table's 64 bits and fp64's angle are exact next to that for positions below 2^20; then one rounding to the type
    bound = torch.zeros_like(y)
    bound[..., a] = bound[..., b] = 8 * 2.0 ** -24 * size * (xa.abs() + xb.abs())
    u = torch.finfo(x.dtype).eps / 2
    bound[..., :R] += u * y[..., :R].abs() + torch.finfo(x.dtype).smallest_normal * u
    return y, bound

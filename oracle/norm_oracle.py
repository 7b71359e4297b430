"""Layer norm by its formula in 64 bits (CPU), with bounds on what rounding may do to a kernel's results.

Test infrastructure only."""
from __future__ import annotations

import torch

E = 2.0 ** -24
CHAIN = 64          # additions one after the other in a row's sum, at most: 32 in a thread, 6 between lanes, 16 between waves


def rounding(x, dtype):
    """Half a step of the type at x, and of its subnormal numbers."""
    info = torch.finfo(dtype)
    return info.eps / 2 * x.abs() + info.smallest_normal * info.eps / 2


def layer_norm(s, w=None, b=None, eps=1e-5, gy=None, gs=None):
    """{name: (result in fp64, how far each element may be off before it is rounded)} of y and, with its gradient gy, dx, dw, db.
    s [rows, D], w and b [D] or None; gs: gradient of s itself.

    A row's sums are off by CHAIN * e of the sum of their terms' sizes.  The mean is subtracted in two steps, the second of which
    takes away what the rounding of the first left, so that a difference d is off by its own roundings and the second sum's, not by
    the mean's; what is left of the first in the variance is far below it (rows up to 10^4 spreads from zero), which a factor of
    two in the variance's bound covers.  h = d * inv is then off by E_h = e ((CHAIN + 12) |h| + (CHAIN + 4) mean|h|).  dw and db
    are sums over the rows in fp32."""
    s = s.double()
    rows, D = s.shape
    w64 = torch.ones(D, dtype=torch.float64) if w is None else w.double()
    b64 = torch.zeros(D, dtype=torch.float64) if b is None else b.double()
    d = s - s.mean(-1, keepdim=True)
    inv = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * inv
    e_h = E * ((CHAIN + 12) * h.abs() + (CHAIN + 4) * h.abs().mean(-1, keepdim=True))
    y = h * w64 + b64
    out = {}
    out["y"] = y, e_h * w64.abs() + 3 * E * ((h * w64).abs() + b64.abs())
    if gy is not None:
        g = gy.double()
        a = g * w64
        s1, s2 = a.mean(-1, keepdim=True), (a * h).mean(-1, keepdim=True)
        e1 = (CHAIN + 2) * E * a.abs().mean(-1, keepdim=True)
        e2 = (CHAIN + 3) * E * (a * h).abs().mean(-1, keepdim=True) + (a.abs() * e_h).mean(-1, keepdim=True)
        inner = a - s1 - h * s2
        size = a.abs() + s1.abs() + (h * s2).abs()
        e_in = 5 * E * size + e1 + h.abs() * e2 + e_h * s2.abs()
        dx = inv * inner
        e_dx = inv * (e_in + (CHAIN + 12) * E * inner.abs())
        if gs is not None:
            dx = dx + gs.double()
            e_dx = e_dx + 2 * E * gs.double().abs()
        out["dx"] = dx, e_dx
        out["dw"] = (g * h).sum(0), (g.abs() * e_h).sum(0) + (rows + 64) * E * (g * h).abs().sum(0)
        out["db"] = g.sum(0), (rows + 64) * E * g.abs().sum(0)
    return out

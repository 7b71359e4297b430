"""Rotary positions of the decoder's queries and keys on the HIP kernel (``amoe_rotary``).

Pair i of a head turns by position * theta_i, theta_i = base^(-2 i / dim).  The pairs are (i, i + dim / 2), or (2 i, 2 i + 1) when
interleaved; elements behind the first ``dim`` of a head stay.  For contexts past the trained one the angles are scaled:

  "linear"  theta / factor: positions squeezed into the trained range;
  "base"    base * factor^(dim / (dim - 2)): the slowest pair is stretched by ``factor``, the fastest keeps its angle;
  "parts"   pairs that turn 32 times or more within ``trained_context`` keep their angle, those that turn once or less are
            stretched by ``factor``, those between in proportion; turned values grow by 1 + 0.1 ln(factor).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor, nn

from . import _abi, ops, raw

SCALINGS = ("none", "linear", "base", "parts")


def _angles(dim: int, base: float, scaling: str, factor: float, trained_context: Optional[int]):
    """Radians per position of every pair."""
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    theta = [base ** (-2.0 * i / dim) for i in range(dim // 2)]
    if scaling == "linear":
        theta = [t / factor for t in theta]
    elif scaling == "parts":
        keep = [min(1.0, max(0.0, (trained_context * t / (2 * math.pi) - 1) / 31)) for t in theta]
        theta = [t * (w + (1 - w) / factor) for t, w in zip(theta, keep)]
    return theta


def _turns(theta) -> Tensor:
    """Revolutions per position times 2^64, as the int64 with those bits: what the kernel multiplies positions by, exactly."""
    words = [round(t / (2 * math.pi) * 2 ** 64) % 2 ** 64 for t in theta]
    return torch.tensor([w - 2 ** 64 if w >= 2 ** 63 else w for w in words], dtype=torch.int64)


def _rows(t: Tensor) -> Tensor:
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _dims(t: Tensor):
    """(stride, size) of the dimensions in which t has more than one element, the widest stride first."""
    return sorted(((st, n) for n, st in zip(t.shape, t.stride()) if n > 1), reverse=True)


def _reach(dims) -> int:
    return 1 + sum(st * (n - 1) for st, n in dims)


def _apart(a: Tensor, b: Tensor) -> bool:
    """Whether two tensors of one type share no element, as far as their strides show it: one lies behind the other, or both
    stay within their own part of every period of some stride that all wider ones are multiples of."""
    x, y = _dims(a), _dims(b)
    off = (b.data_ptr() - a.data_ptr()) // a.element_size()
    if off >= _reach(x) or -off >= _reach(y):
        return True
    for m, _ in {*x, *y}:
        if m and not any(st % m for st, _ in (*x, *y) if st >= m):
            at = off % m
            if _reach([d for d in x if d[0] < m]) <= at and at + _reach([d for d in y if d[0] < m]) <= m:
                return True
    return False


def _check_out(q: Tensor, k: Tensor, oq: Tensor, ok: Tensor) -> None:
    if oq.numel() + ok.numel() == 0:
        return
    for o in (oq, ok):
        dims = _dims(o)
        if any(st < _reach(dims[i + 1:]) for i, (st, _) in enumerate(dims)):
            raise ValueError("out must have memory of its own for every element")
    for o, t, own in ((oq, q, True), (ok, k, True), (oq, k, False), (ok, q, False), (oq, ok, False)):
        in_place = own and o.data_ptr() == t.data_ptr() and all(n == 1 or a == b for n, a, b in zip(o.shape, o.stride(), t.stride()))
        if o.numel() and t.numel() and not in_place and not _apart(o, t):
            raise ValueError("out must be the inputs element for element, or have memory apart from them and from each other")


def rotate(q: Tensor, k: Tensor, turns: Tensor, positions: Optional[Tensor] = None, start: int = 0, interleaved: bool = False,
           size: float = 1.0, inverse: bool = False, out: Optional[Tuple[Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor]:
    """q [B, S, H, d] and k [B, S, G, d] turned by their positions (``amoe_rotary``), into new tensors or into ``out``, whose
    strides are free but for adjacent head elements: q and k themselves, or memory apart from them, such as the rows of a cache
    at which all its sequences go on.  turns: int64 [dim / 2], as ``Rotary`` holds it; inverse: the other way round."""
    ops._need_gpu(q, k, turns, positions)
    shape, kv = q.shape, k.shape
    if len(shape) != 4 or len(kv) != 4:
        raise ValueError("q and k must be [batch, tokens, heads, head size]")
    B, S, H, d = shape
    if kv[0] != B or kv[1] != S or kv[3] != d:
        raise ValueError(f"q {tuple(shape)} and k {tuple(kv)} do not match")
    dtype, device = q.dtype, q.device
    code = raw.code_of(dtype)
    if k.dtype != dtype:
        raise TypeError("q and k must share one dtype")
    if turns.dtype != torch.int64 or turns.dim() != 1 or not turns.is_contiguous():
        raise TypeError("turns must be a contiguous int64 vector")
    R = 2 * turns.numel()
    if not 2 <= R <= d:
        raise ValueError(f"{R} turning elements do not fit heads of {d}")
    if k.device != device or turns.device != device or (positions is not None and positions.device != device):
        raise ValueError("all tensors must be on one device")
    place, place64, pb, ps = 0, False, 0, 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, not {positions.dtype}")
        if start:
            raise ValueError("positions or start, not both")
        place, place64 = positions.data_ptr(), positions.dtype == torch.int64
        if positions.shape == (B, S):
            pb, ps = positions.stride()
        elif positions.shape == (S,):
            ps = positions.stride(0)
        else:
            raise ValueError(f"positions must be [{S}] or [{B}, {S}], not {tuple(positions.shape)}")
    q, k = _rows(q), _rows(k)
    if out is None:
        oq, ok = q.new_empty(shape), k.new_empty(kv)
    else:
        oq, ok = out
        ops._need_gpu(oq, ok)
        for t, o in ((q, oq), (k, ok)):
            if o.shape != t.shape or o.dtype != dtype or o.device != device or (o.stride(3) != 1 and d > 1):
                raise ValueError("out must have the shapes, dtype and device of q and k, with adjacent head elements")
        _check_out(q, k, oq, ok)
    sq, sk, tq, tk = q.stride(), k.stride(), oq.stride(), ok.stride()
    args = _abi.ROTARY_ARGS.pack(
        code, B, S, H, kv[2], d, R, interleaved, inverse, size, turns.data_ptr(), place, place64, pb, ps, start,
        q.data_ptr(), sq[0], sq[1], sq[2], k.data_ptr(), sk[0], sk[1], sk[2],
        oq.data_ptr(), tq[0], tq[1], tq[2], ok.data_ptr(), tk[0], tk[1], tk[2])
    lib = ops.get_lib()
    with ops.device_of(q):
        rc = lib.amoe_rotary(args, ops._stream(q))
    if rc:
        _abi.check(lib, rc, "amoe_rotary")
    if out is not None:
        # (a backward pass that saved them is to notice; inference tensors have no versions)
        torch.autograd.graph.increment_version([t for t in out if not t.is_inference()])
    return oq, ok


class RotaryFunction(torch.autograd.Function):
    """The gradient of a turn is the turn the other way round, itself differentiable in the same way."""

    @staticmethod
    def forward(ctx, q, k, turns, positions, start, interleaved, size, inverse):
        ctx.save_for_backward(turns, positions)
        ctx.args = (start, interleaved, size, not inverse)
        return rotate(q, k, turns, positions, start, interleaved, size, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        turns, positions = ctx.saved_tensors
        f = RotaryFunction.apply if torch.is_grad_enabled() else rotate
        return (*f(gq, gk, turns, positions, *ctx.args), None, None, None, None, None, None)


class RotaryInto(torch.autograd.Function):
    """``rotate`` into tensors that are there, for whom something watches: no derivative of either mode."""

    @staticmethod
    def forward(ctx, q, k, oq, ok, turns, positions, start, interleaved, size):
        ctx.mark_dirty(oq, ok)
        return rotate(q, k, turns, positions, start, interleaved, size, out=(oq, ok))


class Rotary(nn.Module):
    """``rotary(q, k, positions=None, start=0) -> (q, k)`` turned.  positions: int32 / int64 [S] or [B, S], any value; without
    them token s stands at start + s.  The table is an int64 buffer, so that ``.to(torch.bfloat16)`` of a model leaves the
    angles as they are.  ``out``: tensors to write to instead (without gradients only)."""

    def __init__(self, dim: int, base: float = 10000.0, interleaved: bool = False, scaling: str = "none", factor: float = 1.0,
                 trained_context: Optional[int] = None):
        super().__init__()
        if dim < 2 or dim % 2 or dim > 2048:
            raise ValueError(f"the turning part of a head has 2 to 2048 elements, an even number, not {dim}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling must be one of {SCALINGS}, not {scaling!r}")
        if not base >= 1.0 or not factor >= 1.0 or math.isinf(base) or math.isinf(factor):
            raise ValueError("base and factor must be finite and at least 1")
        if scaling == "parts" and (trained_context is None or trained_context < 1):
            raise ValueError("scaling by parts needs the trained context")
        self.dim, self.interleaved = dim, interleaved
        self.size = 1.0 + 0.1 * math.log(factor) if scaling == "parts" else 1.0
        self.register_buffer("turns", _turns(_angles(dim, base, scaling, factor, trained_context)), persistent=False)

    def forward(self, q: Tensor, k: Tensor, positions: Optional[Tensor] = None, start: int = 0,
                out: Optional[Tuple[Tensor, Tensor]] = None) -> Tuple[Tensor, Tensor]:
        args = (q, k, self.turns, positions, start, self.interleaved, self.size)
        grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad)
        if out is not None:
            if grad or any(t.requires_grad for t in out):
                raise RuntimeError("out is for calls without gradients")
            if torch.compiler.is_compiling() or torch._C._get_tracing_state() is not None:
                torch.ops.amoe.rotary_into(q, k, *out, *args[2:])
                return out
            return rotate(*args, out=out) if ops.unwatched() else RotaryInto.apply(q, k, *out, *args[2:])
        if torch.compiler.is_compiling():
            return torch.ops.amoe.rotary(*args, False)
        if not grad and ops.unwatched():
            return rotate(*args)
        return RotaryFunction.apply(*args, False)

    def extra_repr(self) -> str:
        return f"dim={self.dim}, interleaved={self.interleaved}"


from . import library  # noqa: E402,F401  (registers the operators that traced calls go through; it imports this module)

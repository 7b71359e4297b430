"""Layer norm of the decoder on the HIP kernels (``amoe_layer_norm_fwd`` / ``_bwd``), with the residual sum before it.

``s = x + residual`` (rounded to the type), ``y = (s - mean) / sqrt(var + eps) * weight + bias`` over the last dimension; a row is
read once, and the backward pass leaves one gradient of s for both summands.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch
from torch import Tensor, nn

from . import _abi, ops, raw
from .attention import once

MAX_WIDTH = 32768


def _check(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
    """(weight, bias) as vectors that the library takes, the types' codes, rows and their elements."""
    ops._need_gpu(x, residual, weight, bias)
    shape, dtype, device = x.shape, x.dtype, x.device
    code = wcode = raw.code_of(dtype)
    if not shape or not 1 <= shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rows have 1 to {MAX_WIDTH} elements, not {tuple(shape)[-1:]}")
    D = shape[-1]
    if residual is not None and (residual.shape != shape or residual.dtype != dtype or residual.device != device):
        raise ValueError("residual must have x's shape, dtype and device")
    if not 0.0 <= eps <= 3e38:
        raise ValueError(f"eps must be a finite number of 0 or more, not {eps}")
    if weight is not None:
        weight, wcode = _vector(weight, D, dtype, device, "weight"), raw.code_of(weight.dtype)
    if bias is not None:
        bias = _vector(bias, D, dtype, device, "bias")
        if weight is None:
            wcode = raw.code_of(bias.dtype)
        elif bias.dtype != weight.dtype:
            raise TypeError("weight and bias must share one dtype")
    return weight, bias, code, wcode, x.numel() // D, D


def _vector(t: Tensor, D: int, dtype: torch.dtype, device: torch.device, name: str) -> Tensor:
    if t.shape != (D,):
        raise ValueError(f"{name} must be [{D}], not {tuple(t.shape)}")
    if t.dtype != dtype and t.dtype != torch.float32:
        raise TypeError(f"{name} must be {dtype} or float32, not {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, x on {device}")
    return t if t.is_contiguous() else t.contiguous()


def _ptr(t: Optional[Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _rows(t: Tensor, D: int):
    """(what has to live until the launch, its address, elements from row to row): views are calls into torch, most tensors need none."""
    if t.is_contiguous():
        return t, t.data_ptr(), D
    t = ops._rows2d(t)
    return t, t.data_ptr(), t.stride(0)


def layer_norm_forward(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
                       residual: Optional[Tensor] = None,
                       want_stats: bool = False) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """(y, s, stats [rows, 3] fp32): ``amoe_layer_norm_fwd``.  s is None without a residual (it is x), stats without want_stats."""
    weight, bias, code, wcode, n, D = _check(x, residual, weight, bias, eps)
    shape = x.shape
    x, xp, xl = _rows(x, D)
    y = x.new_empty(shape)
    s = stats = None
    rp = rl = 0
    if residual is not None:
        residual, rp, rl = _rows(residual, D)
        s = x.new_empty(shape)
    if want_stats:
        stats = x.new_empty((n, 3), dtype=torch.float32)
    lib = ops.get_lib()
    args = _abi.NORM_ARGS.pack(code, wcode, n, D, eps, xp, xl, _ptr(weight), _ptr(bias), _ptr(stats), rp, rl,
                               y.data_ptr(), _ptr(s), 0, 0, 0, 0, 0, 0, 0)
    with ops.device_of(x):
        rc = lib.amoe_layer_norm_fwd(args, ops._stream(x))
    if rc:
        _abi.check(lib, rc, "amoe_layer_norm_fwd")
    return y, s, stats


@functools.lru_cache(maxsize=1024)
def _workspace(lib, code: int, n: int, D: int) -> int:
    """Bytes of ``amoe_layer_norm_bwd_workspace`` with a gradient of the weight or bias: the sizes decide, not where tensors are."""
    return lib.amoe_layer_norm_bwd_workspace(_abi.NORM_ARGS.pack(code, code, n, D, 0.0, *[0] * 14, 8, 0))


def layer_norm_backward(gy: Tensor, s: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], stats: Tensor, gs: Optional[Tensor] = None,
                        want_x: bool = True, want_weight: bool = True, want_bias: bool = True):
    """(gradient of s, of weight, of bias) from those of y and (gs) of s itself: ``amoe_layer_norm_bwd``; None for what is not
    wanted or not there."""
    weight, bias, code, wcode, n, D = _check(s, gs, weight, bias, 0.0)
    shape = s.shape
    if gy.shape != shape or gy.dtype != s.dtype or gy.device != s.device:
        raise ValueError("the gradient must have s's shape, dtype and device")
    if stats.shape != (n, 3) or stats.dtype != torch.float32 or stats.device != s.device:
        raise ValueError(f"stats must be fp32 [{n}, 3] on {s.device}")
    stats = stats if stats.is_contiguous() else stats.contiguous()
    dx = s.new_empty(shape) if want_x else None
    want_weight, want_bias = want_weight and weight is not None, want_bias and bias is not None
    if n == 0:
        return dx, torch.zeros_like(weight) if want_weight else None, torch.zeros_like(bias) if want_bias else None
    dw = torch.empty_like(weight) if want_weight else None
    db = torch.empty_like(bias) if want_bias else None
    s, sp, sl = _rows(s, D)
    gy, yp, yl = _rows(gy, D)
    gp = gl = 0
    if gs is not None:
        gs, gp, gl = _rows(gs, D)
    lib = ops.get_lib()
    args = _abi.NORM_ARGS.pack(code, wcode, n, D, 0.0, sp, sl, _ptr(weight), _ptr(bias), stats.data_ptr(), 0, 0, 0, 0,
                               yp, yl, gp, gl, _ptr(dx), _ptr(dw), _ptr(db))
    need = _workspace(lib, code, int(n), int(D)) if want_weight or want_bias else 0
    with ops.device_of(s):
        ws = s.new_empty(need, dtype=torch.uint8) if need else None
        rc = lib.amoe_layer_norm_bwd(args, _ptr(ws), need, ops._stream(s))
    if rc:
        _abi.check(lib, rc, "amoe_layer_norm_bwd")
    return dx, dw, db


class LayerNormFunction(torch.autograd.Function):
    """(y, s) of a sum, y alone of x."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps):
        y, s, stats = layer_norm_forward(x, weight, bias, eps, residual, want_stats=True)
        ctx.save_for_backward(x if s is None else s, weight, bias, stats)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    def backward(ctx, gy, gs=None):
        s, weight, bias, stats = ctx.saved_tensors
        need = ctx.needs_input_grad
        if gy is None:                       # (only the sum was used)
            grads = gs, None if weight is None else torch.zeros_like(weight), None if bias is None else torch.zeros_like(bias)
        else:
            grads = layer_norm_backward(gy, s, weight, bias, stats, gs, need[0] or need[1], need[2], need[3])
        if torch.is_grad_enabled():
            grads = once(grads, "layer norm")
        dx, dw, db = grads
        return dx if need[0] else None, dx if need[1] else None, dw if need[2] else None, db if need[3] else None, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5,
               residual: Optional[Tensor] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Layer norm over the last dimension of x; with residual (y, s), s = x + residual rounded to their type and y its norm: the sum
    that the next block adds to.  x and residual of different types are both taken in the wider one.

    Float32, bfloat16 or float16, rows of 1 to 32768 elements, any strides with adjacent elements of a row (others are copied);
    weight and bias [D] of x's type or float32, each optional.  Sums are formed in fp32, the mean as if in more (rows far from
    zero keep their spread); the squares of what differs from the mean, itself as sums in fp32 give it, and their sum have to stay finite in
    fp32 (elements up to 2^70 that differ by up to 2^55 do).  Differentiable once in all four; equal inputs give equal bits in both
    directions."""
    if residual is not None and residual.dtype != x.dtype:
        wide = torch.promote_types(x.dtype, residual.dtype)
        x, residual = x.to(wide), residual.to(wide)
    if torch.compiler.is_compiling():
        y, s, _ = torch.ops.amoe.layer_norm_fwd(x, residual, weight, bias, eps)
        return y if residual is None else (y, s)
    if ops.unwatched() and not (torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)
                                                             or (weight is not None and weight.requires_grad)
                                                             or (bias is not None and bias.requires_grad))):
        y, s, _ = layer_norm_forward(x, weight, bias, eps, residual)
        return y if s is None else (y, s)
    return LayerNormFunction.apply(x, residual, weight, bias, eps)


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` of the last dimension on these kernels, with its parameters and state dict: ``norm(x)``, or
    ``norm(x, residual) -> (y, x + residual)``.  Autocast changes nothing here: y is of x's type (of the wider one with a residual), where
    ``nn.LayerNorm`` gives float32.  Parameters are of y's type or float32: those of a 16-bit module are refused with a float32 stream."""

    def __init__(self, width: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None, dtype=None):
        if not isinstance(width, int) or not 1 <= width <= MAX_WIDTH:
            raise ValueError(f"rows have 1 to {MAX_WIDTH} elements, not {width}")
        super().__init__(width, eps, elementwise_affine, bias, device, dtype)

    def forward(self, x: Tensor, residual: Optional[Tensor] = None):
        return layer_norm(x, self.weight, self.bias, self.eps, residual)


from . import library  # noqa: E402,F401  (registers the operators that traced calls go through; it imports this module)

"""Softmax attention of the decoder on the HIP kernels: training (forward and backward) and new tokens over a cache.

The reference's decoder is the third-party ``sigma_moe`` model (example_aihwkit.py:6, 86-100); these operators stand beside the
expert layer in ``decoder.py``.  ``out = softmax(scale * q k^T + mask) v`` in one pass over the keys; the backward pass makes the
probabilities again from each row's log-sum, so nothing of size queries x keys is ever stored.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _abi, ops, raw

MAX_HEAD = 128


def _rows(t: Tensor) -> Tensor:
    """A [B, rows, heads, d] operand whose heads are adjacent elements."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _marks(t: Optional[Tensor], B: int, like: Tensor, name: str) -> Optional[Tensor]:
    if t is None:
        return None
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    if t.shape != (B,):
        raise ValueError(f"{name} must hold one value per sequence, [{B}], not {tuple(t.shape)}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, q on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _check(q: Tensor, k: Tensor, v: Tensor) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("q, k and v must be [batch, tokens, heads, head size]")
    raw.dtype_code(q)
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError("q, k and v must share one dtype")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on one device")
    if k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not match")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"{q.shape[2]} query heads cannot share {k.shape[2]} key heads evenly")
    if not 1 <= q.shape[3] <= MAX_HEAD:
        raise ValueError(f"heads have 1 to {MAX_HEAD} elements, not {q.shape[3]}")


def _scale(scale: Optional[float], d: int) -> float:
    if scale is None:
        return 1.0 / math.sqrt(d)
    if not 0.0 < scale < 3.4e38:
        raise ValueError(f"scale must be positive and finite, not {scale}")
    return float(scale)


def _pack(q, k, v, lengths, starts, causal, scale, out, lse, go=None, grads=(0, 0, 0)) -> bytes:
    B, S, H, d = q.shape
    return _abi.ATTN_ARGS.pack(
        raw.dtype_code(q), B, S, k.shape[1], H, k.shape[2], d, causal, scale,
        q.data_ptr(), *q.stride()[:3], k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3],
        0 if lengths is None else lengths.data_ptr(), lengths is not None and lengths.dtype == torch.int64,
        0 if starts is None else starts.data_ptr(), starts is not None and starts.dtype == torch.int64,
        out.data_ptr(), 0 if lse is None else lse.data_ptr(),
        *((0, 0, 0, 0) if go is None else (go.data_ptr(), *go.stride()[:3])), *grads)


def attention_forward(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None,
                      causal: bool = True, scale: Optional[float] = None,
                      want_lse: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """(out [B, S, H, d], lse [B, H, S] fp32 or None): ``amoe_attention_fwd``.  lse is what ``attention_backward`` reads."""
    ops._need_gpu(q, k, v, lengths, starts)
    _check(q, k, v)
    scale = _scale(scale, q.shape[3])
    q, k, v = _rows(q), _rows(k), _rows(v)
    B, S, H, d = q.shape
    lengths, starts = _marks(lengths, B, q, "lengths"), _marks(starts, B, q, "starts")
    lib = ops.get_lib()
    out = torch.empty((B, S, H, d), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, S), dtype=torch.float32, device=q.device) if want_lse else None
    args = _pack(q, k, v, lengths, starts, causal, scale, out, lse)
    with ops.device_of(q):
        need = lib.amoe_attention_fwd_workspace(args)
        ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
        rc = lib.amoe_attention_fwd(args, None if ws is None else ws.data_ptr(), need, ops._stream(q))
    _abi.check(lib, rc, "amoe_attention_fwd")
    return out, lse


def attention_backward(go: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, lengths: Optional[Tensor] = None,
                       starts: Optional[Tensor] = None, causal: bool = True, scale: Optional[float] = None,
                       want_kv: bool = True) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """(dq, dk, dv) of ``attention_forward``'s arguments and results (``amoe_attention_bwd``); without want_kv only dq."""
    ops._need_gpu(go, q, k, v, out, lse, lengths, starts)
    _check(q, k, v)
    scale = _scale(scale, q.shape[3])
    if go.shape != q.shape or out.shape != q.shape or go.dtype != q.dtype or out.dtype != q.dtype:
        raise ValueError("out and its gradient must have q's shape and dtype")
    B, S, H, d = q.shape
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, S) or any(t.device != q.device for t in (go, out, lse)):
        raise ValueError("lse must be fp32 [batch, heads, queries], and all tensors on one device")
    q, k, v, go = _rows(q), _rows(k), _rows(v), _rows(go)
    out, lse = out.contiguous(), lse.contiguous()
    lengths, starts = _marks(lengths, B, q, "lengths"), _marks(starts, B, q, "starts")
    lib = ops.get_lib()
    dq = torch.empty((B, S, H, d), dtype=q.dtype, device=q.device)
    dk = dv = None
    if want_kv:
        dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
    args = _pack(q, k, v, lengths, starts, causal, scale, out, lse, go,
                 (dq.data_ptr(), 0 if dk is None else dk.data_ptr(), 0 if dv is None else dv.data_ptr()))
    with ops.device_of(q):
        ws = torch.empty(max(lib.amoe_attention_bwd_workspace(args), 4), dtype=torch.uint8, device=q.device)
        rc = lib.amoe_attention_bwd(args, ws.data_ptr(), ws.numel(), ops._stream(q))
    _abi.check(lib, rc, "amoe_attention_bwd")
    return dq, dk, dv


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, starts, causal, scale):
        out, lse = attention_forward(q, k, v, lengths, starts, causal, scale, want_lse=True)
        ctx.save_for_backward(q, k, v, lengths, starts, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, lengths, starts, out, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv = attention_backward(go, q, k, v, out, lse, lengths, starts, ctx.causal, ctx.scale, need[1] or need[2])
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = True, scale: Optional[float] = None,
              lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None) -> Tensor:
    """Attention of q [B, S, H, d] over k, v [B, T, G, d] -> [B, S, H, d]; H is a multiple of G, and query head h reads key head
    h // (H // G).  Float32, bfloat16 or float16, heads of 1 to 128 elements, any strides with adjacent head elements (others
    are copied).

    lengths [B] (int32 / int64): sequence b holds the keys [0, lengths[b]); those behind are not read, whatever lies there.
    causal: query i stands at position starts[b] + i (starts None: T - S + i, the last S of T) and sees keys up to its own
    position.  scale: 1 / sqrt(d) unless given.  A query that sees no key gives zeros and zero gradients; so do keys that a
    sequence does not hold.  k and v may be a cache with room behind what it holds; a single query per sequence over a long
    one is split along the keys.  Differentiable once in q, k and v; equal inputs give equal bits in both directions."""
    if torch.compiler.is_compiling():
        want = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
        return torch.ops.amoe.attention_fwd(q, k, v, lengths, starts, causal, scale, want)[0]
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) and ops.unwatched():
        return attention_forward(q, k, v, lengths, starts, causal, scale)[0]
    return Attention.apply(q, k, v, lengths, starts, causal, scale)


from . import library  # noqa: E402,F401  (registers the operators that traced calls go through; it imports this module)

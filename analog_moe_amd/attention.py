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

from . import _abi, ops, raw

MAX_HEAD = 128


def _rows(t: Tensor) -> Tensor:
    """A [B, rows, heads, d] operand whose heads are adjacent elements."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _marks(t: Tensor, B: int, device: torch.device, name: str) -> Tensor:
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, not {t.dtype}")
    if t.shape != (B,):
        raise ValueError(f"{name} must hold one value per sequence, [{B}], not {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, q on {device}")
    return t if t.is_contiguous() else t.contiguous()


class _Call:
    """One call's operands, checked, as the library takes them.  (Made for every call: kept lean.)"""
    __slots__ = ("q", "k", "v", "lengths", "starts", "head", "middle", "shape", "kv_shape")

    def __init__(self, q, k, v, lengths, starts, causal, scale):
        ops._need_gpu(q, k, v, lengths, starts)
        shape, kv = q.shape, k.shape
        if len(shape) != 4 or len(kv) != 4:
            raise ValueError("q, k and v must be [batch, tokens, heads, head size]")
        B, S, H, d = shape
        T, G = kv[1], kv[2]
        dtype, device = q.dtype, q.device
        code = raw.code_of(dtype)
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError("q, k and v must share one dtype")
        if k.device != device or v.device != device:
            raise ValueError("q, k and v must be on one device")
        if kv != v.shape or kv[0] != B or kv[3] != d:
            raise ValueError(f"q {tuple(shape)}, k {tuple(kv)} and v {tuple(v.shape)} do not match")
        if G == 0 or H == 0 or H % G:
            raise ValueError(f"{H} query heads cannot share {G} key heads evenly")
        if not 1 <= d <= MAX_HEAD:
            raise ValueError(f"heads have 1 to {MAX_HEAD} elements, not {d}")
        if scale is None:
            scale = 1.0 / math.sqrt(d)
        elif not 2.0 ** -126 <= scale <= 2.0 ** 127:
            raise ValueError(f"scale must be from 2^-126 to 2^127, not {scale}")
        q, k, v = _rows(q), _rows(k), _rows(v)
        n = m = n64 = m64 = 0
        if lengths is not None:
            lengths = _marks(lengths, B, device, "lengths")
            n, n64 = lengths.data_ptr(), lengths.dtype == torch.int64
        if starts is not None:
            starts = _marks(starts, B, device, "starts")
            m, m64 = starts.data_ptr(), starts.dtype == torch.int64
        self.q, self.k, self.v, self.lengths, self.starts, self.shape, self.kv_shape = q, k, v, lengths, starts, shape, kv
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        self.head = (code, B, S, T, H, G, d, causal, scale, q.data_ptr(), qs[0], qs[1], qs[2], k.data_ptr(), ks[0], ks[1], ks[2],
                     v.data_ptr(), vs[0], vs[1], vs[2], n, n64, m, m64)

    def pack(self, out: Tensor, lse: Optional[Tensor], rest: Optional[Tensor], go: Optional[Tensor] = None, grads=(0, 0, 0)) -> bytes:
        gp, gs = (0, (0, 0, 0)) if go is None else (go.data_ptr(), go.stride())
        return _abi.ATTN_ARGS.pack(*self.head, out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                                   0 if rest is None else rest.data_ptr(), gp, gs[0], gs[1], gs[2], *grads)

    def forward(self, want_lse: bool):
        q, lib = self.q, ops.get_lib()
        out = q.new_empty(self.shape)
        lse = rest = None
        if want_lse:
            B, S, H, _ = self.shape
            lse = q.new_empty((B, H, S), dtype=torch.float32)
            rest = None if q.dtype == torch.float32 else q.new_empty(self.shape)
        args = self.pack(out, lse, rest)
        with ops.device_of(q):
            need = lib.amoe_attention_fwd_workspace(args)
            ws = q.new_empty(need, dtype=torch.uint8) if need else None
            rc = lib.amoe_attention_fwd(args, None if ws is None else ws.data_ptr(), need, ops._stream(q))
        if rc:
            _abi.check(lib, rc, "amoe_attention_fwd")
        return out, lse, rest

    def backward(self, go: Tensor, out: Tensor, lse: Tensor, rest: Optional[Tensor], want_kv: bool):
        q, lib, go = self.q, ops.get_lib(), _rows(go)
        dq = q.new_empty(self.shape)
        dk = dv = None
        if want_kv:
            dk, dv = q.new_empty(self.kv_shape), q.new_empty(self.kv_shape)
            args = self.pack(out, lse, rest, go, (dq.data_ptr(), dk.data_ptr(), dv.data_ptr()))
        else:
            args = self.pack(out, lse, rest, go, (dq.data_ptr(), 0, 0))
        with ops.device_of(q):
            ws = q.new_empty(max(lib.amoe_attention_bwd_workspace(args), 4), dtype=torch.uint8)
            rc = lib.amoe_attention_bwd(args, ws.data_ptr(), ws.numel(), ops._stream(q))
        if rc:
            _abi.check(lib, rc, "amoe_attention_bwd")
        return dq, dk, dv


def attention_forward(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None,
                      causal: bool = True, scale: Optional[float] = None,
                      want_lse: bool = False) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """(out [B, S, H, d], lse [B, H, S] fp32, rest like out): ``amoe_attention_fwd``.  With want_lse lse and, for 16-bit types,
    rest (what the rounding of out took away) are there for ``attention_backward``, else None."""
    return _Call(q, k, v, lengths, starts, causal, scale).forward(want_lse)


def attention_backward(go: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, rest: Optional[Tensor] = None,
                       lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None, causal: bool = True,
                       scale: Optional[float] = None, want_kv: bool = True) -> Tuple[Tensor, Optional[Tensor], Optional[Tensor]]:
    """(dq, dk, dv) of ``attention_forward``'s arguments and results (``amoe_attention_bwd``); without want_kv only dq."""
    ops._need_gpu(go, out, lse, rest)
    call = _Call(q, k, v, lengths, starts, causal, scale)
    B, S, H, _ = call.shape
    if go.shape != call.shape or out.shape != call.shape or go.dtype != q.dtype or out.dtype != q.dtype:
        raise ValueError("out and its gradient must have q's shape and dtype")
    if lse.dtype != torch.float32 or tuple(lse.shape) != (B, H, S) or any(t.device != q.device for t in (go, out, lse)):
        raise ValueError("lse must be fp32 [batch, heads, queries], and all tensors on one device")
    if rest is not None:
        if rest.shape != call.shape or rest.dtype != q.dtype or rest.device != q.device:
            raise ValueError("rest must have out's shape, dtype and device")
        rest = rest.contiguous()
    return call.backward(go, out.contiguous(), lse.contiguous(), rest, want_kv)


class Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, starts, causal, scale):
        out, lse, rest = _Call(q, k, v, lengths, starts, causal, scale).forward(True)
        ctx.save_for_backward(q, k, v, lengths, starts, out, lse, rest)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    def backward(ctx, go):
        q, k, v, lengths, starts, out, lse, rest = ctx.saved_tensors
        need = ctx.needs_input_grad
        # (what the forward pass left may come back through hooks in another layout)
        out, lse, rest = (t if t is None or t.is_contiguous() else t.contiguous() for t in (out, lse, rest))
        dq, dk, dv = _Call(q, k, v, lengths, starts, ctx.causal, ctx.scale).backward(go, out, lse, rest, need[1] or need[2])
        grads = dq if need[0] else None, dk if need[1] else None, dv if need[2] else None
        if torch.is_grad_enabled():
            grads = once(grads, "attention")
        return (*grads, None, None, None, None)


def once(grads, what: str):
    """Gradients of a backward pass that is itself differentiated (create_graph): going back through them is an error, not
    a gradient that silently lacks a term."""
    error = torch._C._functions.DelayedError(f"{what} is differentiable once: its backward pass has no derivative", 1)
    return tuple(None if g is None else error(g.detach().requires_grad_()) for g in grads)


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = True, scale: Optional[float] = None,
              lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None) -> Tensor:
    """Attention of q [B, S, H, d] over k, v [B, T, G, d] -> [B, S, H, d]; H is a multiple of G, and query head h reads key head
    h // (H // G).  Float32, bfloat16 or float16, heads of 1 to 128 elements, any strides with adjacent head elements (others
    are copied).

    lengths [B] (int32 / int64): sequence b holds the keys [0, lengths[b]); those behind are not read, whatever lies there.
    causal: query i stands at position starts[b] + i (starts None: T - S + i, the last S of T) and sees keys up to its own
    position.  scale: 1 / sqrt(d) unless given, from 2^-126 to 2^127.  A query that sees no key gives zeros and zero gradients;
    so do keys that a sequence does not hold.  k and v may be a cache with room behind what it holds; a single query per
    sequence over a long one is split along the keys.  Differentiable once in q, k and v; equal inputs give equal bits in both
    directions.  Scores may be of any finite size.  Heads of whole 16-byte chunks (multiples of 8 elements, 4 in float32) at
    aligned addresses run several times faster than others.

    An element that is infinite or not a number in a key or value that the sequence holds, in a query or in its gradient, may
    reach every result of that sequence and head: a masked score's probability is zero, and its products are formed, as in the
    formula.  Capturing a backward pass: as elsewhere in torch, no graph of the same leaves from outside the capture may be alive."""
    if torch.compiler.is_compiling():
        want = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
        return torch.ops.amoe.attention_fwd(q, k, v, lengths, starts, causal, scale, want)[0]
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)) and ops.unwatched():
        return attention_forward(q, k, v, lengths, starts, causal, scale)[0]
    return Attention.apply(q, k, v, lengths, starts, causal, scale)


def shared_attention_forward(q: Tensor, k: Tensor, v: Tensor, prefix_k: Tensor, prefix_v: Tensor, lengths: Optional[Tensor] = None,
                             starts: Optional[Tensor] = None, prefix_lengths: Optional[Tensor] = None, causal: bool = True,
                             scale: Optional[float] = None) -> Tensor:
    """``amoe_attention_shared_fwd``; ``shared_attention`` describes it."""
    ops._need_gpu(prefix_k, prefix_v, prefix_lengths)
    call = _Call(q, k, v, lengths, starts, causal, scale)
    code, B, S, T, H, G, d, causal, scale, *rest = call.head
    shape = prefix_k.shape
    if len(shape) != 4 or shape != prefix_v.shape or shape[2] != G or shape[3] != d:
        raise ValueError(f"prefix_k {tuple(shape)} and prefix_v {tuple(prefix_v.shape)} do not match k {tuple(call.kv_shape)}")
    if prefix_k.dtype != q.dtype or prefix_v.dtype != q.dtype:
        raise TypeError("q, k, v and the prefix must share one dtype")
    if prefix_k.device != q.device or prefix_v.device != q.device:
        raise ValueError("q, k, v and the prefix must be on one device")
    N, P = shape[:2]
    if B and (N == 0 or B % N):
        raise ValueError(f"{B} sequences cannot continue {N} prefixes evenly")
    pk, pv = _rows(prefix_k), _rows(prefix_v)
    n = n64 = 0
    if prefix_lengths is not None:
        prefix_lengths = _marks(prefix_lengths, N, q.device, "prefix_lengths")
        n, n64 = prefix_lengths.data_ptr(), prefix_lengths.dtype == torch.int64
    out = q.new_empty(call.shape)
    ks, vs = pk.stride(), pv.stride()
    args = _abi.SHARED_ATTN_ARGS.pack(code, B, S, T, P, N, H, G, d, causal, scale, *rest[:12], pk.data_ptr(), ks[0], ks[1], ks[2],
                                      pv.data_ptr(), vs[0], vs[1], vs[2], *rest[12:], n, n64, out.data_ptr())
    lib = ops.get_lib()
    with ops.device_of(q):
        need = lib.amoe_attention_shared_fwd_workspace(args)
        ws = q.new_empty(need, dtype=torch.uint8) if need else None
        rc = lib.amoe_attention_shared_fwd(args, None if ws is None else ws.data_ptr(), need, ops._stream(q))
    if rc:
        _abi.check(lib, rc, "amoe_attention_shared_fwd")
    return out


def shared_attention(q: Tensor, k: Tensor, v: Tensor, prefix_k: Tensor, prefix_v: Tensor, *, causal: bool = True,
                     scale: Optional[float] = None, lengths: Optional[Tensor] = None, starts: Optional[Tensor] = None,
                     prefix_lengths: Optional[Tensor] = None) -> Tensor:
    """``attention`` of q [B, S, H, d] over the keys of a prefix [N, P, G, d], then the sequence's own k, v [B, T, G, d]: every B / N
    sequences in a row continue one prefix, which is read once for all of them.

    All queries see the first prefix_lengths[n] keys of their prefix (None: P).  Own keys are as in ``attention``: lengths, starts
    and the causal mask count among them (query i of sequence b sees own keys up to starts[b] + i; starts None: T - S + i).  T and P may
    be 0.  A query that sees no key gives zeros.  For serving: no gradients."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, prefix_k, prefix_v)):
        raise RuntimeError("shared_attention has no gradient: call it under torch.no_grad()")
    if torch.compiler.is_compiling() or not ops.unwatched():
        return torch.ops.amoe.attention_shared(q, k, v, prefix_k, prefix_v, lengths, starts, prefix_lengths, causal, scale)
    return shared_attention_forward(q, k, v, prefix_k, prefix_v, lengths, starts, prefix_lengths, causal, scale)


from . import library  # noqa: E402,F401  (registers the operators that traced calls go through; it imports this module)

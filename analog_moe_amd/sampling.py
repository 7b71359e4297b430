"""The choice of the decoder's next token on the HIP kernel (``amoe_sample``): temperature, top-k, top-p and min-p, from given numbers.

Random numbers are inputs, so that a draw can be repeated, checked and captured into a graph: fill ``u`` in place (``u.uniform_()``)
before every replay.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
from torch import Tensor

from . import _abi, ops, raw

MAX_VOCABULARY = (1 << 20) - 1

Setting = Union[float, Tensor]


def _setting(v, shape, device, name: str, types, low: float, high: float):
    """(tensor or None, address, number for all)."""
    if isinstance(v, Tensor):
        if v.dtype not in types:
            raise TypeError(f"{name} must be {' or '.join(str(t) for t in types)}, not {v.dtype}")
        if v.shape != shape:
            raise ValueError(f"{name} must be a number or hold one per row, {tuple(shape)}, not {tuple(v.shape)}")
        if v.device != device:
            raise ValueError(f"{name} is on {v.device}, logits on {device}")
        v = v if v.is_contiguous() else v.contiguous()
        return v, v.data_ptr(), low
    if not low <= v <= high:
        raise ValueError(f"{name} must be from {low} to {high}, not {v}")
    return None, 0, v


_F32, _INT = (torch.float32,), (torch.int32, torch.int64)
_MOST = 3.4028234663852886e38


def draw(logits: Tensor, u: Tensor, temperature: Setting = 1.0, top_k: Union[int, Tensor] = 0, top_p: Setting = 1.0, min_p: Setting = 0.0,
         want_logprob: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """(ids, logprob or None): ``amoe_sample``; ``sample`` describes it."""
    ops._need_gpu(logits, u, *(t for t in (temperature, top_k, top_p, min_p) if isinstance(t, Tensor)))
    code = raw.code_of(logits.dtype)
    if logits.dim() < 1 or not 1 <= logits.shape[-1] <= MAX_VOCABULARY:
        raise ValueError(f"rows have 1 to {MAX_VOCABULARY} logits, not {tuple(logits.shape)[-1:]}")
    shape, device, V = logits.shape[:-1], logits.device, logits.shape[-1]
    if u.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"u must be float32 or float64, not {u.dtype}")
    if u.shape != shape or u.device != device:
        raise ValueError(f"u must hold one number per row, {tuple(shape)} on {device}")
    u = u if u.is_contiguous() else u.contiguous()
    t, tp, t_all = _setting(temperature, shape, device, "temperature", _F32, 0.0, _MOST)
    k, kp, k_all = _setting(top_k, shape, device, "top_k", _INT, 0, 2 ** 63 - 1)
    p, pp, p_all = _setting(top_p, shape, device, "top_p", _F32, 0.0, 1.0)
    m, mp, m_all = _setting(min_p, shape, device, "min_p", _F32, 0.0, 1.0)
    if not hasattr(k_all, "__index__"):
        raise TypeError(f"top_k must be an integer, not {k_all}")
    rows = ops._rows2d(logits)
    n = rows.shape[0]
    ids = torch.empty(shape, dtype=torch.int64, device=device)
    logprob = torch.empty(shape, dtype=torch.float32, device=device) if want_logprob else None
    lib = ops.get_lib()
    args = _abi.SAMPLE_ARGS.pack(code, n, V, rows.data_ptr(), rows.stride(0), u.data_ptr(), u.dtype == torch.float64, tp, pp, mp, kp,
                                 k is not None and k.dtype == torch.int64, t_all, p_all, m_all, k_all, ids.data_ptr(),
                                 0 if logprob is None else logprob.data_ptr())
    with ops.device_of(logits):
        need = lib.amoe_sample_workspace(args)
        ws = rows.new_empty(need, dtype=torch.uint8) if need else None
        rc = lib.amoe_sample(args, None if ws is None else ws.data_ptr(), need, ops._stream(logits))
    if rc:
        _abi.check(lib, rc, "amoe_sample")
    return ids, logprob


def sample(logits: Tensor, u: Tensor, temperature: Setting = 1.0, top_k: Union[int, Tensor] = 0, top_p: Setting = 1.0,
           min_p: Setting = 0.0, want_logprob: bool = False) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """One token of each row of logits [..., V] (float32, bfloat16 or float16), by u [...] (float32 or float64, from [0, 1)): int64 ids
    [...], and with want_logprob the float32 logarithms of their probabilities among what was kept.

    With weight_i = exp((logit_i - largest) / temperature), tokens ranked by their logits and the lower index first among equals:
    kept are the first top_k (0: all), of these the shortest run from the top with at least top_p of their weight (the first one
    always), of these what weighs min_p of the largest or more.  The token is the first, in the order of the indices, up to which the
    kept ones weigh more than u times all of them.  Temperature 0: the largest logit, with logarithm 0.  Settings are numbers, or
    tensors with one for each row (float32; top_k int32 / int64), which are taken as the nearest that is allowed.

    Not-a-numbers count as minus infinity, which is never drawn; a row of nothing else gives -1 and minus infinity.  Weights are whole
    multiples of 2^-44 of the largest (what weighs less than half of that is never drawn, and weights that differ by less are equal) and
    sums of them exact, so that a token is the same every time; it is the definition's unless u or top_p meets a border between tokens to
    within V times 2^-44 of the largest weight, or min_p a weight to within 2^-44.  Numbers are taken in float32.  Up to 2^20 - 1 logits a
    row.  No gradients."""
    if want_logprob and torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("the logarithms of sample have no gradient: call it under torch.no_grad(), or on detached logits")
    if torch.compiler.is_compiling() or not ops.unwatched():
        def split(v, none):
            return (v, none) if isinstance(v, Tensor) else (None, v)
        (t, ta), (k, ka), (p, pa), (m, ma) = split(temperature, 0.0), split(top_k, 0), split(top_p, 0.0), split(min_p, 0.0)
        ids, logprob = torch.ops.amoe.sample(logits.detach(), u, t, k, p, m, ta, ka, pa, ma)
    else:
        ids, logprob = draw(logits, u, temperature, top_k, top_p, min_p, want_logprob)
    return (ids, logprob) if want_logprob else ids


from . import library  # noqa: E402,F401  (registers the operators that traced calls go through; it imports this module)

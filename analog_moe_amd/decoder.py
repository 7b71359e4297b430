"""A minimal SigmaMoE decoder: the caller of the CVMM path in the full training step.

The reference's example trains ``sigma_moe.SigmaMoEForCausalLM`` (example_aihwkit.py:6, 86-100), a
third-party model whose feed-forward blocks are the SigmaMoE layers this package implements.  That model is
not part of the reference checkout; this module provides the smallest stand-in that exercises the layer the
same way: token + position embedding, pre-norm blocks of causal self-attention and an analog SigmaMoE
feed-forward, final norm and language-model head.  Embeddings are stock PyTorch; the
MoE feed-forward is ``AnalogSigmaMoELayer`` (or any module with its ``forward(x) -> (y, reg_loss)``).  Attention is stock
PyTorch with a learned position table, or, with ``rotary``, this package's attention and rotary positions, which also
serve: prompts and single tokens over a ``KVCache``, sequences of different lengths in one batch, several that continue one
prompt, tokens drawn from the logits (``generate``).  Norms are ``nn.LayerNorm``, or, with ``norm=LayerNorm`` of this package, its
kernels, which form the sum with the residual stream too.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Optional, Tuple

import torch
import torch.nn.functional as F
from torch import Tensor, nn

from .attention import attention, shared_attention
from .norm import LayerNorm
from .rotary import Rotary
from .sampling import sample


class CausalSelfAttention(nn.Module):
    def __init__(self, d_model: int, n_heads: int):
        super().__init__()
        if d_model % n_heads:
            raise ValueError("d_model must be a multiple of n_heads")
        self.n_heads = n_heads
        self.qkv = nn.Linear(d_model, 3 * d_model, bias=False)
        self.proj = nn.Linear(d_model, d_model, bias=False)

    def forward(self, x: Tensor) -> Tensor:
        B, S, D = x.shape
        q, k, v = self.qkv(x).view(B, S, 3, self.n_heads, D // self.n_heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v, is_causal=True)
        return self.proj(a.transpose(1, 2).reshape(B, S, D))


@dataclass
class KVCache:
    """Keys (turned) and values of every layer with room for ``keys.shape[2]`` tokens a sequence.  held: int64 [batch], the
    tokens that each sequence holds; most: no sequence holds more.

    A step of single tokens captured into a graph keeps the tensors and the number it was captured with: set ``most`` to the room
    less one before, so that it reads keys up to the end, and advance the tensor that ``held`` was before the call, in place and
    within the capture:

        held, cache.most = cache.held, cache.keys.shape[2] - 1
        with torch.cuda.graph(graph):
            logits, _ = model(token, cache=cache)
            held.add_(1)

    and replay no further than the room (past it the positions are an assertion on the device).

    prefix: a cache that every batch / (its batch) sequences in a row continue (``share``); held and most count what comes after it."""
    keys: Tensor                                 # [layers, batch, room, key heads, head size]
    values: Tensor
    held: Tensor
    most: int = 0
    prefix: Optional["KVCache"] = None

    def share(self, copies: int, room: int) -> "KVCache":
        """An empty cache for ``copies`` sequences after each of this one's, with room for ``room`` tokens of their own: what this one
        holds now is read where it is, for all of them at once.  This one may go on by itself, but its tokens must stay."""
        if self.prefix is not None:
            raise ValueError("a cache that continues another one is not shared again")
        if copies < 1 or room < 0:
            raise ValueError(f"{copies} sequences with room for {room} tokens")
        layers, batch, _, heads, head = self.keys.shape
        keys, values = (t.new_empty((layers, batch * copies, room, heads, head)) for t in (self.keys, self.values))
        held = self.held.new_zeros(batch * copies)
        return KVCache(keys, values, held, 0, KVCache(self.keys, self.values, self.held.clone(), self.most))


class RotarySelfAttention(nn.Module):
    """Causal self-attention with rotary positions; every n_heads / kv_heads heads share keys and values."""

    def __init__(self, d_model: int, n_heads: int, kv_heads: int, rotary: Rotary):
        super().__init__()
        if d_model % n_heads or n_heads % kv_heads:
            raise ValueError("d_model must be a multiple of n_heads, and n_heads of kv_heads")
        self.n_heads, self.kv_heads, self.head = n_heads, kv_heads, d_model // n_heads
        if rotary.dim > self.head:
            raise ValueError(f"rotary positions turn {rotary.dim} elements of heads of {self.head}")
        self.rotary = rotary
        self.qkv = nn.Linear(d_model, (n_heads + 2 * kv_heads) * self.head, bias=False)
        self.proj = nn.Linear(d_model, d_model, bias=False)

    def forward(self, x: Tensor, lengths: Optional[Tensor] = None, cache: Optional[KVCache] = None, layer: int = 0,
                positions: Optional[Tensor] = None, places: Optional[Tensor] = None) -> Tensor:
        """lengths: tokens of each sequence that are not padding; with a cache, tokens held when x's are in it, positions [B, S]
        where x's stand, and places [B, S] where they stand in the cache (None: there too)."""
        B, S, D = x.shape
        q, k, v = self.qkv(x).view(B, S, -1, self.head).split((self.n_heads, self.kv_heads, self.kv_heads), dim=2)
        q, k = self.rotary(q, k, positions)
        starts = None
        if cache is not None:
            at = (torch.arange(B, device=x.device)[:, None], positions if places is None else places)
            keys, values = cache.keys[layer], cache.values[layer]
            keys.index_put_(at, k.to(keys.dtype))
            values.index_put_(at, v.to(values.dtype))
            k, v, starts = keys[:, :cache.most + S], values[:, :cache.most + S], cache.held
        # (a cache of another type than q's: attention in the cache's)
        if cache is not None and cache.prefix is not None:
            pk, pv = (t[layer, :, :cache.prefix.most] for t in (cache.prefix.keys, cache.prefix.values))
            out = shared_attention(q.to(k.dtype), k, v, pk, pv, lengths=lengths, starts=starts, prefix_lengths=cache.prefix.held).to(q.dtype)
        else:
            out = attention(q.to(k.dtype), k, v, lengths=lengths, starts=starts).to(q.dtype)
        return self.proj(out.reshape(B, S, D))


class DecoderBlock(nn.Module):
    def __init__(self, d_model: int, n_heads: int, ffn: nn.Module, attn: Optional[nn.Module] = None,
                 norm: Callable[[int], nn.Module] = nn.LayerNorm):
        super().__init__()
        self.ln_attn = norm(d_model)
        self.attn = CausalSelfAttention(d_model, n_heads) if attn is None else attn
        self.ln_ffn = norm(d_model)
        self.ffn = ffn

    @property
    def sums(self) -> bool:
        """Whether its norms form the sums with the residual stream."""
        return isinstance(self.ln_attn, LayerNorm) and isinstance(self.ln_ffn, LayerNorm)

    def forward(self, x: Tensor, add: Optional[Tensor] = None, split: bool = False, **attn_args):
        """(stream, regularisation); split, with norms that form the sums: on the stream x + add (None: x), and (stream, what is to be
        added to it, regularisation)."""
        if split:
            n, x = (self.ln_attn(x), x) if add is None else self.ln_attn(add, x)
            n, x = self.ln_ffn(self.attn(n, **attn_args), x)
            return x, *self.ffn(n)
        x = x + self.attn(self.ln_attn(x), **attn_args)
        y, reg = self.ffn(self.ln_ffn(x))
        return x + y, reg


class SigmaMoEDecoder(nn.Module):
    """``make_ffn(layer_index) -> module`` builds the feed-forward of each block.  rotary: positions and attention of this
    package instead of a learned table of ``context`` positions and stock attention; kv_heads (None: n_heads) of its heads
    hold keys and values.  norm: ``nn.LayerNorm``, or ``analog_moe_amd.norm.LayerNorm`` (the same parameters)."""

    def __init__(self, vocab_size: int, d_model: int, n_layers: int, n_heads: int, context: int,
                 make_ffn: Callable[[int], nn.Module], rotary: Optional[Rotary] = None, kv_heads: Optional[int] = None,
                 norm: Callable[[int], nn.Module] = nn.LayerNorm):
        super().__init__()
        if kv_heads is not None and rotary is None:
            raise ValueError("kv_heads goes with rotary: stock attention has as many key heads as heads")
        self.tok = nn.Embedding(vocab_size, d_model)
        self.pos = nn.Embedding(context, d_model) if rotary is None else None

        def attn():
            return None if rotary is None else RotarySelfAttention(d_model, n_heads, kv_heads or n_heads, rotary)
        self.blocks = nn.ModuleList(DecoderBlock(d_model, n_heads, make_ffn(i), attn(), norm) for i in range(n_layers))
        self.ln_out = norm(d_model)
        self.head = nn.Linear(d_model, vocab_size, bias=False)

    def new_cache(self, batch: int, room: int) -> KVCache:
        """An empty cache for ``batch`` sequences of up to ``room`` tokens, of the model's device and type (under autocast: of the
        type that it makes keys and values in)."""
        if self.pos is not None:
            raise ValueError("a cache goes with rotary positions")
        attn, like = self.blocks[0].attn, self.head.weight
        shape = (len(self.blocks), batch, room, attn.kv_heads, attn.head)
        kind = like.device.type
        dtype = torch.get_autocast_dtype(kind) if torch.is_autocast_enabled(kind) else like.dtype
        keys, values = (torch.empty(shape, dtype=dtype, device=like.device) for _ in range(2))
        return KVCache(keys, values, torch.zeros(batch, dtype=torch.int64, device=like.device))

    def forward(self, ids: Tensor, labels: Optional[Tensor] = None, reg_weight: float = 0.0,
                lengths: Optional[Tensor] = None, cache: Optional[KVCache] = None):
        """Logits [B, S, V] and the summed regularisation loss of the MoE layers; with ``labels`` the scalar
        training loss (cross-entropy in fp32 + reg_weight * regularisation) instead of the logits.

        With rotary positions: lengths [B], the tokens of each sequence of ids that are not padding (which stands behind
        them; give such labels as -100).  cache: ids follow what it holds, and it holds them afterwards (without gradients)."""
        B, S = ids.shape
        x = self.tok(ids)
        args = {}
        if self.pos is not None:
            if lengths is not None or cache is not None:
                raise ValueError("lengths and a cache go with rotary positions")
            x = x + self.pos(torch.arange(S, device=ids.device))
        elif cache is None:
            args = dict(lengths=lengths)
        else:
            if torch.is_grad_enabled():
                raise RuntimeError("a cache is filled without gradients: call the decoder under torch.no_grad()")
            if cache.keys.shape[1] != B or cache.most + S > cache.keys.shape[2]:
                raise ValueError(f"{B} sequences of {S} more tokens do not fit a cache of {cache.keys.shape[1]} with room for "
                                 f"{cache.keys.shape[2]}, {cache.most} taken")
            # (within what ids have: positions past the cache's room are an assertion on the device)
            held = cache.held + (S if lengths is None else lengths.clamp(0, S))
            args = dict(lengths=held, cache=cache, positions=cache.held[:, None] + torch.arange(S, device=ids.device))
            if cache.prefix is not None:
                before = cache.prefix.held.repeat_interleave(B // cache.prefix.held.shape[0], output_size=B)
                args.update(places=args["positions"], positions=args["positions"] + before[:, None])
        reg = x.new_zeros((), dtype=torch.float32)
        split, add = isinstance(self.ln_out, LayerNorm) and all(blk.sums for blk in self.blocks), None
        for i, blk in enumerate(self.blocks):
            if cache is not None:
                args["layer"] = i
            if split:
                x, add, r = blk(x, add, True, **args)
            else:
                x, r = blk(x, **args)
            reg = reg + r.float()
        if cache is not None:
            cache.held, cache.most = held, cache.most + S
        logits = self.head(self.ln_out(x) if add is None else self.ln_out(add, x)[0])
        if labels is None:
            return logits, reg
        loss = F.cross_entropy(logits.float().view(B * S, -1), labels.reshape(-1))
        return loss + reg_weight * reg, reg

    @torch.no_grad()
    def generate(self, ids: Tensor, steps: int, copies: int = 1, lengths: Optional[Tensor] = None,
                 generator: Optional[torch.Generator] = None, want_logprob: bool = False, **settings):
        """``steps`` tokens after each prompt of ids [N, S] (lengths [N]: the tokens of each that are not padding, at least one), drawn
        ``copies`` times: int64 [N * copies, steps], those of one prompt in a row; with want_logprob also the float32 logarithms of
        their probabilities.  settings: temperature, top_k, top_p, min_p of ``sample`` (tensors hold one per sequence); temperature 0
        makes all copies the same.  The prompts' keys are kept and read once for all copies."""
        N, S = ids.shape
        if S < 1 or steps < 0 or copies < 1:
            raise ValueError(f"{steps} tokens after {copies} copies of prompts of {S}")
        if lengths is not None:
            lengths = lengths.clamp(1, S)
        cache = self.new_cache(N, S if copies > 1 else S + steps)
        logits, _ = self(ids, lengths=lengths, cache=cache)
        last = logits[:, -1] if lengths is None else logits[torch.arange(N, device=ids.device), lengths.long() - 1]
        if copies > 1:
            cache, last = cache.share(copies, steps), last.repeat_interleave(copies, 0)
        tokens = torch.empty(N * copies, steps, dtype=torch.int64, device=ids.device)
        logprob = torch.empty(N * copies, steps, dtype=torch.float32, device=ids.device)
        for s in range(steps):
            u = torch.rand(N * copies, generator=generator, device=ids.device)
            tokens[:, s], logprob[:, s] = sample(last, u, want_logprob=True, **settings)
            if s + 1 < steps:
                # (a row without a number has no token: -1 is not to be looked up)
                logits, _ = self(tokens[:, s:s + 1].clamp_min(0), cache=cache)
                last = logits[:, -1]
        return (tokens, logprob) if want_logprob else tokens

    def post_update_step(self) -> None:
        """Weight clipping of the analog layers after an optimizer step (moe_layer_aihwkit_lightning.py:509-517)."""
        for blk in self.blocks:
            if hasattr(blk.ffn, "post_update_step"):
                blk.ffn.post_update_step()

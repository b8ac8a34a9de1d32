"""Attention of a block's tokens to an encoder's states of another length.

``cross_attention(q, k, v, key_lengths=..., key_mask=...)`` is ``flash_attention(q, k, v,
k_lens=context_lens)`` of the reference's WanT2VCrossAttention (reference/livewan_wan21/wan/modules/model.py) on
kernels of this package: q [B, Lq, H, D] from the block's q linear, k and v [B, Lk, Hk, D] from the text's or
image's k / v linears, of any two lengths (Lq = Lk is the block's self-attention). Keys beyond a sample's
length or masked out do not count, whatever they hold; a query without keys gets zeros, and so do its gradients.
Query heads may share key heads (H a multiple of Hk). Gradients of q, k and v, summed in a fixed order.

bf16: scores, softmax and sums in float32; the weights are rounded to bf16 for their product with v, as they and dS
are in the backward of a sample of more than 2^30 products (heads, rows, keys and channels multiplied; below, both
enter in two parts, to 16 bits, whatever the batch). delta is formed from the rounded output, but from float32 weights
where a sample has at most 64 keys that count. float32: float32 throughout, on the fp32 matrix core.
"""
from __future__ import annotations

import functools
import math

import torch

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)


def _fail(message: str) -> None:
    raise RuntimeError("cross attention: " + message)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if kernels.attention_layout(t):
        return t
    t = t.contiguous()
    return t if kernels.attention_layout(t) else t.clone()


class CrossAttentionFunction(torch.autograd.Function):
    """``apply(q, k, v, key_lengths, key_mask, scale)`` -> out."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, key_mask, scale: float):
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        out, lse = kernels.cross_attention(q, k, v, key_lengths=key_lengths, key_mask=key_mask, scale=scale, checked=True)
        ctx.save_for_backward(q, k, v, out, lse, key_lengths, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @kernels.first_order
    def backward(ctx, g):
        q, k, v, out, lse, key_lengths, key_mask = ctx.saved_tensors
        grads = kernels.cross_attention_backward(q, k, v, out, lse, _aligned(g if g.dtype is q.dtype else g.to(q.dtype)),
                                                 key_lengths=key_lengths, key_mask=key_mask, scale=ctx.scale, checked=True)
        return (*[d if want else None for d, want in zip(grads, ctx.needs_input_grad)], None, None, None)


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.dtype, t.device)


# What a call's shapes, types and options allow, checked once per combination of them.
@functools.lru_cache(maxsize=256)
def _plan(q, k, v, key_lengths, key_mask, scale) -> float:
    for name, (shape, dtype, device) in (("q", q), ("k", k), ("v", v)):
        if len(shape) != 4:
            _fail(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(shape)}")
        if dtype not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {dtype}")
        if dtype != q[1] or device != q[2]:
            _fail("q, k and v share one dtype and device")
    B, _, H, D = q[0]
    Lk, Hk = k[0][1:3]
    if k[0] != v[0] or k[0][0] != B or k[0][3] != D:
        _fail(f"k and v must be [{B}, tokens, heads, {D}], got {tuple(k[0])} and {tuple(v[0])}")
    if Hk < 1 or H < 1 or H % Hk:
        _fail(f"{H} query heads do not share {Hk} key heads evenly")
    if D % 8 or not 8 <= D <= 128:
        _fail(f"head_dim must be a multiple of 8 up to 128, got {D}")
    scale = D ** -0.5 if scale is None else scale
    if not (math.isfinite(scale) and scale > 0):
        _fail("scale must be positive")
    if key_lengths is not None:
        shape, dtype, device = key_lengths
        if device != q[2] or dtype not in (torch.int32, torch.int64) or tuple(shape) != (B,):
            _fail(f"key_lengths must be int32 or int64 [{B}] on q's device")
    if key_mask is not None:
        shape, dtype, device = key_mask
        if device != q[2] or dtype is not torch.bool or tuple(shape) not in ((Lk,), (1, Lk), (B, Lk)):
            _fail(f"key_mask must be bool [{B}, {Lk}] on q's device")
    if q[2].type != "cuda":
        _fail("the tensors must be ROCm device tensors")
    return scale


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, key_lengths: torch.Tensor | None = None,
                    key_mask: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """softmax(scale q kᵀ) v per head, [B, Lq, H, D] contiguous in q's dtype.

    q [B, Lq, H, D], k and v [B, Lk, Hk, D], bfloat16 or float32, D a multiple of 8 up to 128. key_lengths:
    int32 or int64 [B] on q's device, the number of leading keys that count (clamped to [0, Lk]). key_mask:
    bool [B, Lk] (or [1, Lk], [Lk] for every sample), True where a key counts. scale > 0, 1 / sqrt(D) if not given."""
    if scale is not None:
        scale = kernels.number("scale", scale, _fail)
    scale = _plan(_meta(q), _meta(k), _meta(v), _meta(key_lengths), _meta(key_mask), scale)
    if key_lengths is not None:
        if key_lengths.dtype is torch.int64:
            key_lengths = key_lengths.clamp(0, k.shape[1]).to(torch.int32)
        key_lengths = key_lengths.contiguous()
    if key_mask is not None:
        if key_mask.dim() == 1:
            key_mask = key_mask.unsqueeze(0)
        if not key_mask.is_contiguous() and key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
    if kernels.wants_grad((q, k, v)):
        return CrossAttentionFunction.apply(q, k, v, key_lengths, key_mask, scale)
    return kernels.cross_attention(_aligned(q), _aligned(k), _aligned(v), key_lengths=key_lengths, key_mask=key_mask,
                                   scale=scale, checked=True)[0]

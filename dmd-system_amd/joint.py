"""The joint of two sublayers: the residual stream takes a sublayer's output, the next one's input leaves.

    p  = N_post(y) * post_weight            (or y: most blocks norm only before a sublayer)
    x1 = residual_scale * x + gate * p
    out = N(x1) * m + shift                 m = 1 + scale (a modulation) or scale (a norm's weight)

``gated_residual_norm`` is one kernel forward and one backward (plus the vectors' sums). It covers the three
joints of a Wan block (model.py:298-313: the gate and the affine norm3 after self-attention, no gate and
the modulated norm2 after cross-attention, the gate and the next block's norm1 after the ffn) and blocks
normed on both sides of a sublayer. Unlike the gated GEMM epilogue (``gated_residual``), whose gate is
frozen, every operand has a gradient here, and the next norm needs no pass of its own.
"""
from __future__ import annotations

import functools
import math

import torch

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)


def _fail(message: str) -> None:
    raise RuntimeError("gated residual norm: " + message)


def _laid_out(*tensors):
    return [t if t is None or kernels.rows_layout(t) else kernels.aligned(t) for t in tensors]


class GatedResidualNormFunction(torch.autograd.Function):
    """``apply(x, y, gate, scale, shift, post_weight, cfg)`` -> (x1, out); cfg as _plan gives it."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, post_weight, cfg):
        args = _laid_out(x, y, gate, scale, shift, post_weight)
        ctx.save_for_backward(*args)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        return kernels.joint(*args, **cfg, checked=True)

    @staticmethod
    @kernels.first_order
    def backward(ctx, gx, go):
        if gx is None and go is None:
            return (None,) * 7
        x, y, *vectors = ctx.saved_tensors
        gx = None if gx is None else kernels.aligned(gx if gx.dtype is x.dtype else gx.to(x.dtype))
        go = None if go is None else kernels.aligned(go if go.dtype is y.dtype else go.to(y.dtype))
        grads = kernels.joint_backward(x, y, gx, go, *vectors, **ctx.cfg, want=ctx.needs_input_grad[:6], checked=True)
        return (*grads, None)


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.dtype, t.device)


# What a call's shapes, types and options allow, checked once per combination of them.
@functools.lru_cache(maxsize=256)
def _plan(x, y, gate, scale, shift, post_weight, norm, unit_offset, post_norm, residual_scale, eps) -> dict:
    for name, (shape, dtype, _) in (("x", x), ("y", y)):
        if len(shape) != 3:
            _fail(f"{name} must be [batch, tokens, width], got {tuple(shape)}")
        if dtype not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {dtype}")
    if x[0] != y[0] or x[2] != y[2]:
        _fail(f"x and y share shape and device, got {tuple(x[0])} and {tuple(y[0])}")
    if x[1] is torch.bfloat16 and y[1] is torch.float32:
        _fail("a bfloat16 stream takes a bfloat16 y")
    B, _, W = x[0]
    if W % 8 or not 8 <= W <= 8192:
        _fail(f"width must be a multiple of 8 up to 8192, got {W}")
    if norm not in kernels.NORM_KINDS or (post_norm is not None and post_norm not in kernels.NORM_KINDS):
        _fail("norm and post_norm must be 'layer' or 'rms'")
    if post_weight is not None and post_norm is None:
        _fail("post_weight needs a post_norm")
    if shift is not None and scale is None:
        _fail("a shift needs a scale")
    if not (math.isfinite(eps) and eps > 0):
        _fail("eps must be positive")
    if not math.isfinite(residual_scale):
        _fail("residual_scale must be finite")
    for name, v in (("gate", gate), ("scale", scale), ("shift", shift), ("post_weight", post_weight)):
        if v is None:
            continue
        if v[2] != x[2] or v[1] not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32 on x's device")
        per_sample = name != "post_weight"
        if tuple(v[0]) not in (((W,), (1, W), (B, W), (1, 1, W), (B, 1, W)) if per_sample else ((W,),)):
            _fail(f"{name} must be [{W}]" + (f", [{B}, {W}] or [{B}, 1, {W}]" if per_sample else "") + f", got {tuple(v[0])}")
    if scale is not None and shift is not None and scale[1] != shift[1]:
        _fail("scale and shift share a dtype")
    if x[2].type != "cuda":
        _fail("the tensors must be ROCm device tensors")
    return dict(norm=norm, post=post_norm, unit_offset=unit_offset, alpha=residual_scale, eps=eps)


def gated_residual_norm(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor | None = None,
                        scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, *, norm: str = "layer",
                        unit_offset: bool = True, post_norm: str | None = None,
                        post_weight: torch.Tensor | None = None, residual_scale: float = 1.0,
                        eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """(x1, out) for the residual stream x and a sublayer's output y, [B, T, W] each.

    x1 has x's dtype (bfloat16 or float32), out y's (bfloat16; float32 with a float32 stream). gate, scale
    and shift are per sample ([B, W] or [B, 1, W]) or shared ([W]). norm / post_norm: "layer" or "rms" (both
    with `eps`); without post_norm y joins as it is. unit_offset: out is scaled by 1 + scale (a modulation),
    else by scale (a norm's weight, with shift its bias)."""
    cfg = _plan(_meta(x), _meta(y), _meta(gate), _meta(scale), _meta(shift), _meta(post_weight), norm, bool(unit_offset),
                post_norm, kernels.number("residual_scale", residual_scale, _fail), kernels.number("eps", eps, _fail))
    args = (x, y, gate, scale, shift, post_weight)
    if kernels.wants_grad(args):
        return GatedResidualNormFunction.apply(*args, cfg)
    return kernels.joint(*_laid_out(*args), **cfg, checked=True)

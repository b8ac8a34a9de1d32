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

import math

import torch
from torch.autograd.function import once_differentiable

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)


def _fail(message: str) -> None:
    raise RuntimeError("gated residual norm: " + message)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if kernels.rows_layout(t):
        return t
    t = t.contiguous()
    return t if kernels.rows_layout(t) else t.clone()


class GatedResidualNormFunction(torch.autograd.Function):
    """``apply(x, y, gate, scale, shift, post_weight, cfg)`` -> (x1, out); vectors [B or 1, W] or None."""

    @staticmethod
    def forward(ctx, x, y, gate, scale, shift, post_weight, cfg):
        args = [None if t is None else _aligned(t) for t in (x, y, gate, scale, shift, post_weight)]
        x1, out = kernels.joint(*args, **cfg)
        ctx.save_for_backward(*args)
        ctx.cfg = cfg
        ctx.set_materialize_grads(False)
        return x1, out

    @staticmethod
    @once_differentiable
    def backward(ctx, gx, go):
        if gx is None and go is None:
            return (None,) * 7
        x, y, gate, scale, shift, post_weight = ctx.saved_tensors
        gx = None if gx is None else _aligned(gx.to(x.dtype))
        go = None if go is None else _aligned(go.to(y.dtype))
        grads = kernels.joint_backward(x, y, gx, go, gate, scale, shift, post_weight, **ctx.cfg,
                                       want=ctx.needs_input_grad[:6])
        return (*grads, None)


def _vector(name: str, v: torch.Tensor | None, x: torch.Tensor, per_sample: bool = True) -> torch.Tensor | None:
    """v as [B or 1, W] (a view, so that its gradient comes back in v's own shape)."""
    if v is None:
        return None
    B, _, W = x.shape
    if v.device != x.device or v.dtype not in _DTYPES:
        _fail(f"{name} must be bfloat16 or float32 on x's device")
    if v.dim() == 1 and v.shape[0] == W:
        return v.unsqueeze(0)
    if per_sample and v.dim() == 2 and v.shape[0] in (1, B) and v.shape[1] == W:
        return v
    if per_sample and v.dim() == 3 and v.shape[0] in (1, B) and v.shape[1] == 1 and v.shape[2] == W:
        return v.select(1, 0)
    _fail(f"{name} must be [{W}]" + (f", [{B}, {W}] or [{B}, 1, {W}]" if per_sample else "") + f", got {tuple(v.shape)}")


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
    for name, t in (("x", x), ("y", y)):
        if t.dim() != 3:
            _fail(f"{name} must be [batch, tokens, width], got {tuple(t.shape)}")
        if t.dtype not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {t.dtype}")
    if x.shape != y.shape or x.device != y.device:
        _fail(f"x and y share shape and device, got {tuple(x.shape)} and {tuple(y.shape)}")
    if x.dtype is torch.bfloat16 and y.dtype is torch.float32:
        _fail("a bfloat16 stream takes a bfloat16 y")
    W = x.shape[2]
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
    gate, scale, shift = (_vector(n, v, x) for n, v in (("gate", gate), ("scale", scale), ("shift", shift)))
    post_weight = _vector("post_weight", post_weight, x, per_sample=False)
    if scale is not None and shift is not None and scale.dtype != shift.dtype:
        _fail("scale and shift share a dtype")
    if not x.is_cuda:
        _fail("the tensors must be ROCm device tensors")
    cfg = dict(norm=norm, post=post_norm, unit_offset=bool(unit_offset), alpha=float(residual_scale), eps=float(eps))
    return GatedResidualNormFunction.apply(x, y, gate, scale, shift, post_weight, cfg)

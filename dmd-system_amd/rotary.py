"""Rotary positions with several axes for the heads of q and k, with the RMSNorm in front of them.

A DiT turns the pairs of every head by angles of the token's place in the video: the head's channels
are split over the axes (time, height, width; image models have two), and pair i of an axis of d
channels turns by ``position * theta ** (-2 i / d)``. Wan norms q and k over the whole row first and
pairs neighbouring channels (``rope_apply`` and ``WanSelfAttention.norm_q`` / ``norm_k``,
reference/livewan_wan21/wan/modules/model.py); image models norm each head, some pair the halves.

``rotary_axes_qk(q, k, positions, axis_dims, ...)`` runs both in one launch, ``rotary_axes`` one tensor;
``grid_positions`` builds the positions of (frames, height, width) grids in padded batches. Gradients:
q, k and the norm weights. Outputs are rounded once from float32 arithmetic; angles are formed in 64 bits.
"""
from __future__ import annotations

import math
from typing import Sequence

import torch
from torch.autograd.function import once_differentiable

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)
_PAIRINGS = ("adjacent", "halves")


def _fail(message: str) -> None:
    raise RuntimeError("rotary axes: " + message)


def grid_positions(grid_sizes, tokens: int, device=None, start=0) -> torch.Tensor:
    """int32 [B, tokens, axes]: the coordinates of each sample's grid in row-major order from `start` (a
    number, or one per axis). Tokens behind a sample's grid get the origin, where the rotation leaves
    them as they are.

    grid_sizes: [B, axes] as a tensor (the reference's ``grid_sizes``) or nested sequence."""
    sizes = [[int(v) for v in row] for row in (grid_sizes.tolist() if isinstance(grid_sizes, torch.Tensor) else grid_sizes)]
    if not sizes or not sizes[0] or any(len(r) != len(sizes[0]) for r in sizes):
        _fail("grid_sizes must be [batch, axes]")
    axes = len(sizes[0])
    first = [int(start)] * axes if not isinstance(start, (list, tuple)) else [int(v) for v in start]
    if len(first) != axes:
        _fail(f"start has {len(first)} values for {axes} axes")
    out = torch.zeros(len(sizes), tokens, axes, dtype=torch.int32)
    for b, row in enumerate(sizes):
        n = math.prod(row)
        if min(row) < 0 or n > tokens:
            _fail(f"grid {row} does not fit {tokens} tokens")
        if n:
            grid = torch.meshgrid(*(torch.arange(f, f + s, dtype=torch.int32) for f, s in zip(first, row)), indexing="ij")
            out[b, :n] = torch.stack([g.reshape(-1) for g in grid], dim=1)
    return out.to(device) if device is not None else out


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if kernels.rows_layout(t):
        return t
    t = t.contiguous()
    return t if kernels.rows_layout(t) else t.clone()


def _norm_kinds(name: str, x: torch.Tensor, w: torch.Tensor | None) -> set:
    if w is None:
        return {kernels.NORM_NONE}
    H, D = x.shape[2:]
    if w.device != x.device or w.dtype not in _DTYPES or w.dim() != 1 or w.shape[0] not in (D, H * D):
        _fail(f"{name} must be a bfloat16 or float32 vector of {D} (per head) or {H * D} (the row) on q's device")
    return {kind for kind, n in ((kernels.NORM_ROW, H * D), (kernels.NORM_HEAD, D)) if n == w.shape[0]}


class RotaryAxesFunction(torch.autograd.Function):
    """``apply(positions, axis_dims, theta, halves, norm, eps, n, *tensors, *weights)`` -> n tensors."""

    @staticmethod
    def forward(ctx, positions, axis_dims, theta, halves, norm, eps, n, *args):
        xs, ws = args[:n], args[n:]
        xs = [_aligned(x) for x in xs]
        ws = [_aligned(w) for w in ws] if norm else list(ws)
        ys = kernels.rotary_axes(xs, positions, axis_dims, theta=theta, halves=halves, norm=norm, weights=ws, eps=eps)
        ctx.save_for_backward(positions, *(xs if norm else ()), *(ws if norm else ()))
        ctx.cfg = (axis_dims, theta, halves, norm, eps, n)
        ctx.like = [(x.shape, x.dtype, x.device) for x in xs]
        ctx.set_materialize_grads(False)
        return tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        axis_dims, theta, halves, norm, eps, n = ctx.cfg
        none = (None,) * (7 + 2 * n)
        if all(g is None for g in grads):
            return none
        positions, *saved = ctx.saved_tensors
        xs, ws = (saved[:n], saved[n:]) if norm else (None, [None] * n)
        gs = []
        for g, (shape, dtype, device) in zip(grads, ctx.like):
            g = torch.zeros(shape, dtype=dtype, device=device) if g is None else g.to(dtype)
            gs.append(_aligned(g))
        want_dx, want_dw = ctx.needs_input_grad[7:7 + n], ctx.needs_input_grad[7 + n:]
        dxs, dws = kernels.rotary_axes_backward(xs, gs, positions, axis_dims, theta=theta, halves=halves, norm=norm,
                                                weights=ws, eps=eps, want_dx=want_dx, want_dw=want_dw)
        return (*none[:7], *dxs, *dws)


def _apply(xs, ws, names, positions, axis_dims, theta, pairing, eps):
    first = xs[0]
    for name, x in zip(names, xs):
        if x.dim() != 4:
            _fail(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(x.shape)}")
        if x.dtype not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {x.dtype}")
        if x.dtype != first.dtype or x.device != first.device:
            _fail("q and k share one dtype and device")
        if x.shape[:2] != first.shape[:2] or x.shape[3] != first.shape[3]:
            _fail(f"q and k share batch, tokens and head_dim, got {tuple(first.shape)} and {tuple(x.shape)}")
    B, L, _, D = first.shape
    if D % 16 or not 16 <= D <= 256:
        _fail(f"head_dim must be a multiple of 16 up to 256, got {D}")
    if any(not 1 <= x.shape[2] <= 8192 // D for x in xs):
        _fail(f"heads * head_dim must be between {D} and 8192")
    axis_dims = tuple(int(d) for d in axis_dims)
    if not axis_dims or any(d < 0 or d % 2 for d in axis_dims) or sum(axis_dims) != D:
        _fail(f"axis_dims must be even channel counts that add up to head_dim {D}, got {axis_dims}")
    if pairing not in _PAIRINGS:
        _fail(f"pairing must be one of {_PAIRINGS}, got {pairing!r}")
    if not (math.isfinite(theta) and theta > 0):
        _fail("theta must be positive")
    if not (math.isfinite(eps) and eps > 0):
        _fail("eps must be positive")
    if positions.device != first.device or positions.dtype not in (torch.int32, torch.int64, torch.float32):
        _fail("positions must be int32, int64 or float32 on q's device")
    if positions.requires_grad:
        _fail("positions take no gradient")
    if positions.dim() == 2:
        positions = positions.unsqueeze(0)
    if positions.dim() != 3 or positions.shape[0] not in (1, B) or tuple(positions.shape[1:]) != (L, len(axis_dims)):
        _fail(f"positions must be [{L}, {len(axis_dims)}] or [{B}, {L}, {len(axis_dims)}], got {tuple(positions.shape)}")
    if positions.shape[2] > 1 and positions.stride(2) != 1 or any(s < 0 for s in positions.stride()):
        positions = positions.contiguous()
    if len({w is None for w in ws}) > 1:
        _fail("q_weight and k_weight come together")
    kinds = set.intersection(*(_norm_kinds(f"{name}_weight", x, w) for name, x, w in zip(names, xs, ws)))
    if not kinds:
        _fail("q and k are normed alike: both over the row or both per head")
    if ws[0] is not None and any(w.dtype != ws[0].dtype for w in ws):
        _fail("q_weight and k_weight share a dtype")
    if not first.is_cuda:
        _fail("the tensors must be ROCm device tensors")
    return RotaryAxesFunction.apply(positions, axis_dims, float(theta), pairing == "halves", max(kinds), float(eps),
                                    len(xs), *xs, *ws)


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int], *, theta: float = 10000.0,
                pairing: str = "adjacent", weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x [B, L, H, D] with its heads rotated by `positions` ([L, axes] or [B, L, axes], whole or fractional),
    contiguous and in x's dtype.

    axis_dims: channels of each axis (even, adding up to D), in the order of the positions. pairing:
    "adjacent" turns channels 2i and 2i + 1, "halves" channels i and i + D / 2. weight: RMSNorm first, over the
    token's whole row for [H * D], over each head for [D]."""
    return _apply([x], [weight], ["x"], positions, axis_dims, theta, pairing, eps)[0]


def rotary_axes_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int], *,
                   theta: float = 10000.0, pairing: str = "adjacent", q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_axes of q and k (their head counts may differ) in one launch."""
    return _apply([q, k], [q_weight, k_weight], ["q", "k"], positions, axis_dims, theta, pairing, eps)

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

import functools
import math
from typing import Sequence

import torch

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)
_PAIRINGS = ("adjacent", "halves")


def _fail(message: str) -> None:
    raise RuntimeError("rotary axes: " + message)


def _whole(name: str, value) -> int:
    try:
        whole = int(value)
    except (TypeError, ValueError, OverflowError, RuntimeError):
        _fail(f"{name} must be whole numbers, got a {type(value).__name__}")
    if whole != value:
        _fail(f"{name} must be whole numbers")
    return whole


def grid_positions(grid_sizes, tokens: int, device=None, start=0) -> torch.Tensor:
    """int32 [B, tokens, axes]: the coordinates of each sample's grid in row-major order from `start` (a whole
    number, or one per axis). Tokens behind a sample's grid get the origin, where the rotation leaves
    them as they are.

    grid_sizes: [B, axes] as a tensor (the reference's ``grid_sizes``) or nested sequence."""
    sizes = [[_whole("grid_sizes", v) for v in row] for row in (grid_sizes.tolist() if isinstance(grid_sizes, torch.Tensor) else grid_sizes)]
    if not sizes or not sizes[0] or any(len(r) != len(sizes[0]) for r in sizes):
        _fail("grid_sizes must be [batch, axes]")
    axes = len(sizes[0])
    first = [_whole("start", v) for v in (start if isinstance(start, (list, tuple)) else [start] * axes)]
    if len(first) != axes:
        _fail(f"start has {len(first)} values for {axes} axes")
    out = torch.zeros(len(sizes), tokens, axes, dtype=torch.int32)
    for b, row in enumerate(sizes):
        n = math.prod(row)
        if min(row) < 0 or n > tokens:
            _fail(f"grid {row} does not fit {tokens} tokens")
        if n:
            if min(first) < -2 ** 31 or any(f + s > 2 ** 31 for f, s in zip(first, row)):
                _fail(f"grid {row} from start {first} leaves int32")
            grid = torch.meshgrid(*(torch.arange(f, f + s, dtype=torch.int32) for f, s in zip(first, row)), indexing="ij")
            out[b, :n] = torch.stack([g.reshape(-1) for g in grid], dim=1)
    return out.to(device) if device is not None else out


class RotaryAxesFunction(torch.autograd.Function):
    """``apply(positions, cfg, n, *tensors, *weights)`` -> n tensors; cfg as _plan gives it, no weights without a
    norm."""

    @staticmethod
    def forward(ctx, positions, cfg, n, *args):
        args = [kernels.aligned(t) for t in args]
        xs, ws = args[:n], args[n:]
        ctx.save_for_backward(positions, *(args if ws else ()))
        ctx.cfg, ctx.n = cfg, n
        ctx.like = [(x.shape, x.dtype, x.device) for x in xs]
        ctx.set_materialize_grads(False)
        return tuple(kernels.rotary_axes(xs, positions, weights=ws, checked=True, **cfg))

    @staticmethod
    @kernels.first_order
    def backward(ctx, *grads):
        n, needs = ctx.n, ctx.needs_input_grad
        if all(g is None for g in grads):
            return (None,) * len(needs)
        positions, *saved = ctx.saved_tensors
        gs = []
        for g, (shape, dtype, device) in zip(grads, ctx.like):
            if g is None:
                g = torch.zeros(shape, dtype=dtype, device=device)
            gs.append(kernels.aligned(g if g.dtype is dtype else g.to(dtype)))
        dxs, dws = kernels.rotary_axes_backward(saved[:n] if saved else None, gs, positions, weights=saved[n:],
                                                want_dx=needs[3:3 + n], want_dw=needs[3 + n:], checked=True, **ctx.cfg)
        return (None, None, None, *dxs, *dws)


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.dtype, t.device)


# What a call's shapes, types and options allow, checked once per combination of them.
@functools.lru_cache(maxsize=256)
def _plan(names, xs, ws, positions, axis_dims, theta, pairing, eps) -> dict:
    first, dtype, device = xs[0]
    for name, (shape, dt, dev) in zip(names, xs):
        if len(shape) != 4:
            _fail(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(shape)}")
        if dt not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {dt}")
        if dt != dtype or dev != device:
            _fail("q and k share one dtype and device")
        if shape[:2] != first[:2] or shape[3] != first[3]:
            _fail(f"q and k share batch, tokens and head_dim, got {tuple(first)} and {tuple(shape)}")
    B, L, _, D = first
    if D % 16 or not 16 <= D <= 256:
        _fail(f"head_dim must be a multiple of 16 up to 256, got {D}")
    if any(not 1 <= shape[2] <= 8192 // D for shape, _, _ in xs):
        _fail(f"heads * head_dim must be between {D} and 8192")
    if not axis_dims or any(d < 0 or d % 2 for d in axis_dims) or sum(axis_dims) != D:
        _fail(f"axis_dims must be even channel counts that add up to head_dim {D}, got {axis_dims}")
    if pairing not in _PAIRINGS:
        _fail(f"pairing must be one of {_PAIRINGS}, got {pairing!r}")
    if not (math.isfinite(theta) and theta > 0):
        _fail("theta must be positive")
    if not (math.isfinite(eps) and eps > 0):
        _fail("eps must be positive")
    shape, dt, dev = positions
    if dev != device or dt not in (torch.int32, torch.int64, torch.float32):
        _fail("positions must be int32, int64 or float32 on q's device")
    if tuple(shape) not in ((L, len(axis_dims)), (1, L, len(axis_dims)), (B, L, len(axis_dims))):
        _fail(f"positions must be [{L}, {len(axis_dims)}] or [{B}, {L}, {len(axis_dims)}], got {tuple(shape)}")
    if len({w is None for w in ws}) > 1:
        _fail("q_weight and k_weight come together")
    kinds = {kernels.NORM_NONE} if ws[0] is None else {kernels.NORM_ROW, kernels.NORM_HEAD}
    for name, (shape, _, _), w in zip(names, xs, ws):
        if w is None:
            continue
        H = shape[2]
        if w[2] != device or w[1] not in _DTYPES or tuple(w[0]) not in ((D,), (H * D,)):
            _fail(f"{name}_weight must be a bfloat16 or float32 vector of {D} (per head) or {H * D} (the row) on q's device")
        kinds &= {kind for kind, n in ((kernels.NORM_ROW, H * D), (kernels.NORM_HEAD, D)) if n == w[0][0]}
    if not kinds:
        _fail("q and k are normed alike: both over the row or both per head")
    if ws[0] is not None and any(w[1] != ws[0][1] for w in ws):
        _fail("q_weight and k_weight share a dtype")
    if device.type != "cuda":
        _fail("the tensors must be ROCm device tensors")
    return dict(axis_dims=axis_dims, theta=theta, halves=pairing == "halves", norm=max(kinds), eps=eps)


def _apply(xs, ws, names, positions, axis_dims, theta, pairing, eps):
    if positions.requires_grad:
        _fail("positions take no gradient")
    kernels.refuse_tangents((positions,))
    cfg = _plan(names, tuple([_meta(x) for x in xs]), tuple([_meta(w) for w in ws]), _meta(positions),
                tuple([d if type(d) is int else _whole("axis_dims", d) for d in axis_dims]), kernels.number("theta", theta, _fail), pairing,
                kernels.number("eps", eps, _fail))
    if positions.dim() == 2:
        positions = positions.unsqueeze(0)
    if not positions.is_contiguous() and (positions.stride(2) != 1 or any(s < 0 for s in positions.stride())):
        positions = positions.contiguous()
    args = (*xs, *ws) if cfg["norm"] else xs
    if kernels.wants_grad(args):
        return RotaryAxesFunction.apply(positions, cfg, len(xs), *args)
    args = [kernels.aligned(t) for t in args]
    return tuple(kernels.rotary_axes(args[:len(xs)], positions, weights=args[len(xs):], checked=True, **cfg))


def rotary_axes(x: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int], *, theta: float = 10000.0,
                pairing: str = "adjacent", weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """x [B, L, H, D] with its heads rotated by `positions` ([L, axes] or [B, L, axes], whole or fractional),
    contiguous and in x's dtype.

    axis_dims: channels of each axis (even, adding up to D), in the order of the positions. pairing:
    "adjacent" turns channels 2i and 2i + 1, "halves" channels i and i + D / 2. weight: RMSNorm first, over the
    token's whole row for [H * D], over each head for [D]."""
    return _apply((x,), (weight,), ("x",), positions, axis_dims, theta, pairing, eps)[0]


def rotary_axes_qk(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axis_dims: Sequence[int], *,
                   theta: float = 10000.0, pairing: str = "adjacent", q_weight: torch.Tensor | None = None,
                   k_weight: torch.Tensor | None = None, eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """rotary_axes of q and k (their head counts may differ) in one launch."""
    return _apply((q, k), (q_weight, k_weight), ("q", "k"), positions, axis_dims, theta, pairing, eps)

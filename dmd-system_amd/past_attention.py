"""Attention of a stream's tokens to their own past.

A streaming student generates a clip chunk by chunk (a few latent frames at a time, or token by token): a token attends
to its own chunk and to what was generated before it, mostly to the last chunks (a sliding window) and to the first ones
(sinks), and several samples may continue one past (conditional and unconditional passes, rollouts of one history).

``window_attention(q, k, v, window=..., sinks=..., chunk=...)`` covers whole sequences (training, prompts) and the newest
tokens of a cache; ``prefix_attention(q, k, v, prefix_k, prefix_v, ...)`` adds a prefix that the samples of a group share.
Where they have few tokens each it is read for the rows of all of them together, once per 32 rows (128 where a key head has more
than 64 of them in bf16). Both with gradients of every tensor, the prefix's summed over its samples, all in a fixed order. Query
heads may share key heads (H a multiple of Hk).

A token at position p of a sample with n keys sees the own keys j < min(e, n) with j >= e - window or j < sinks, where
e = (p // chunk + 1) * chunk is the end of its chunk, and all keys of its prefix. Queries that are no token of the sample
(p < 0 or p >= n: padding) get zeros, and so do their gradients, whatever they hold; so do keys behind n. What lies in
k and v where no token of the sample sees it is not used. What is not finite in a token, or in a key that some tokens see, may
reach others in the tiles that hold it, as a product with weight zero does: from v the outputs and from k the dq of rows that do not see
the key (tiles of up to 32 rows and 64 keys), from q and the upstream gradient the dk and dv of keys that the token does not see (tiles
of up to 64 tokens and 32 keys).

The gradients of q, k, v and the prefix are all computed where one is wanted. Saved-tensor hooks may return copies in any layout.
What a call's shapes and strides allow is looked up by them: a cache that grows by slices is planned anew for every length, one of a
fixed size with key_lengths once.

bf16: scores, softmax and sums in float32; the weights are rounded to bf16 for their products (dS too); out is rounded
once, and what that rounding left is kept for the backward (bf16, the size of out). float32: float32 throughout, on
the fp32 matrix core.
"""
from __future__ import annotations

import functools
import math

import torch

from . import kernels

_DTYPES = (torch.bfloat16, torch.float32)
_MOST = 1 << 28  # tokens
_NAMES = ("q", "k", "v", "prefix_k", "prefix_v")


def _fail(message: str) -> None:
    raise RuntimeError("past attention: " + message)


def _whole(name: str, value) -> int:
    if type(value) is int:
        return value
    try:
        whole = int(value)
    except (TypeError, ValueError, OverflowError, RuntimeError):
        _fail(f"{name} must be a whole number, got a {type(value).__name__}")
    if whole != value:
        _fail(f"{name} must be a whole number")
    return whole


def _aligned(t: torch.Tensor) -> torch.Tensor:
    if kernels.attention_layout(t):
        return t
    t = t.contiguous()
    return t if kernels.attention_layout(t) else t.clone()


def _lay_out(call, tensors):
    """(the kernels' plan, the tensors as they take them, their addresses): copies where a layout or an address is not theirs."""
    plan, again = call
    pointers = [t.data_ptr() for t in tensors]
    if plan is None or any([p & 15 for p in pointers]):
        tensors = [_aligned(t) for t in tensors]
        plan, pointers = _planned(tuple([_meta(t) for t in tensors]), again), [t.data_ptr() for t in tensors]
    return plan, tensors, pointers


def _planned(metas, again):
    return _plan(metas, *again)[0]


def _unpack(ctx):
    """(the kernels' plan, what the forward saved, as the plan has it). A saved-tensor hook may return a copy in another layout,
    which is planned again; anything but the tensor it was given is refused."""
    plan, saved = ctx.plan, ctx.saved_tensors
    given = [t for t in saved if t is not None]
    # four short lists: _meta's tuples cost a small backward 3 us more
    if (([t.shape for t in given], [t.dtype for t in given], [t.get_device() for t in given], [t.stride() for t in given]) == plan.given
            and not any([t.data_ptr() & 15 for t in saved[3:]])):
        return plan, saved
    for was, now in zip(plan.metas, [_meta(t) for t in saved]):
        if (was and was[:3]) != (now and now[:3]):
            _fail(f"a saved-tensor hook returned {now and now[:3]} in place of {was and was[:3]}")
    flat = [t if t is None else t.contiguous() for t in saved[:5]]  # the vectors, out and the statistics
    flat = [t if t is None or t.data_ptr() % 16 == 0 else t.clone() for t in flat]
    tensors = [_aligned(t) for t in saved[5:]]
    return _planned(tuple([_meta(t) for t in tensors]), ctx.again), (*flat, *tensors)


class PastAttentionFunction(torch.autograd.Function):
    """``apply(call, key_lengths, query_start, prefix_lengths, q, k, v[, prefix_k, prefix_v])`` -> out; call as _plan
    gives it."""

    @staticmethod
    def forward(ctx, call, key_lengths, query_start, prefix_lengths, *tensors):
        ctx.again = call[1]
        ctx.plan, tensors, pointers = _lay_out(call, tensors)
        out, saved = kernels.past_attention(ctx.plan, tensors, pointers, key_lengths, query_start, prefix_lengths, True)
        ctx.save_for_backward(key_lengths, query_start, prefix_lengths, out, saved, *tensors)
        return out

    @staticmethod
    @kernels.first_order
    def backward(ctx, g):
        plan, (key_lengths, query_start, prefix_lengths, out, saved, *tensors) = _unpack(ctx)
        g = _aligned(g if g.dtype is out.dtype else g.to(out.dtype))
        grads = kernels.past_attention_backward(plan, out, saved, g, tensors, key_lengths, query_start, prefix_lengths)
        return (None, None, None, None, *[d if want else None for d, want in zip(grads, ctx.needs_input_grad[4:])])


def _meta(t: torch.Tensor | None):
    return None if t is None else (t.shape, t.dtype, t.device, t.stride())


def _check_tensors(**tensors) -> None:
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            _fail(f"{name} must be a tensor, got a {type(t).__name__}")


def _check_vector(name: str, meta, n: int, device) -> None:
    if meta is not None:
        shape, dtype, dev, _ = meta
        if dev != device or dtype not in (torch.int32, torch.int64) or tuple(shape) != (n,):
            _fail(f"{name} must be int32 or int64 [{n}] on q's device")


def _layout(shape, strides) -> bool:
    """attention_layout but for the address, which is looked at on every call."""
    return math.prod(shape) == 0 or (
        (shape[3] < 2 or strides[3] == 1) and all([n < 2 or s % 8 == 0 for n, s in zip(shape[:3], strides)])
        and (shape[1] < 2 or strides[1] < kernels.ATTENTION_MAX_STRIDE))


# What a call's shapes, types, strides and options allow, checked once per combination of them: the kernels' plan (None where a
# tensor's layout is not theirs) and what the same call with other tensors is planned from.
@functools.lru_cache(maxsize=512)
def _plan(metas, key_lengths, query_start, prefix_lengths, window, sinks, chunk, scale):
    again = (key_lengths, query_start, prefix_lengths, window, sinks, chunk, scale)
    q, k, v, pk, pv = metas if len(metas) == 5 else (*metas, None, None)
    for name, (shape, dtype, device, _) in (("q", q), ("k", k), ("v", v)):
        if len(shape) != 4:
            _fail(f"{name} must be [batch, tokens, heads, head_dim], got {tuple(shape)}")
        if dtype not in _DTYPES:
            _fail(f"{name} must be bfloat16 or float32, got {dtype}")
        if dtype != q[1] or device != q[2]:
            _fail("q, k and v share one dtype and device")
    (B, Lq, H, D), dtype, device, _ = q
    Lk, Hk = k[0][1:3]
    if k[0] != v[0] or k[0][0] != B or k[0][3] != D:
        _fail(f"k and v must be [{B}, tokens, heads, {D}], got {tuple(k[0])} and {tuple(v[0])}")
    if Hk < 1 or H < 1 or H % Hk:
        _fail(f"{H} query heads do not share {Hk} key heads evenly")
    if D % 8 or not 8 <= D <= 128:
        _fail(f"head_dim must be a multiple of 8 up to 128, got {D}")
    if max(Lq, Lk) > _MOST:
        _fail(f"at most {_MOST} tokens")
    if pk is not None:
        if pk[1:3] != q[1:3] or pv[1:3] != q[1:3]:
            _fail("prefix_k and prefix_v have q's dtype and device")
        if pk[0] != pv[0] or len(pk[0]) != 4 or tuple(pk[0][2:]) != (Hk, D):
            _fail(f"prefix_k and prefix_v must be [tokens, {Hk}, {D}] or [groups, tokens, {Hk}, {D}], got {tuple(pk[0])} and {tuple(pv[0])}")
        if pk[0][0] < 1 or B % pk[0][0]:
            _fail(f"{B} samples do not share {pk[0][0]} prefixes evenly")
        if pk[0][1] > _MOST:
            _fail(f"at most {_MOST} tokens")
        _check_vector("prefix_lengths", prefix_lengths, pk[0][0], device)
    if chunk < 1:
        _fail(f"chunk must be at least 1, got {chunk}")
    if window is not None and window < chunk:
        _fail(f"window must be at least chunk ({chunk}), so that every token sees its own chunk; got {window}")
    if sinks < 0:
        _fail(f"sinks must not be negative, got {sinks}")
    _check_vector("key_lengths", key_lengths, B, device)
    if isinstance(query_start, tuple):
        _check_vector("query_start", query_start, B, device)
    elif query_start is None and Lq > Lk:
        _fail(f"{Lq} queries are no tokens of {Lk} keys: give query_start")
    scale = D ** -0.5 if scale is None else scale
    if not (math.isfinite(scale) and scale > 0):
        _fail("scale must be positive")
    if device.type != "cuda":
        _fail("the tensors must be ROCm device tensors")
    # past these nothing changes, and they fit the kernels' integers
    start = 0 if isinstance(query_start, tuple) else Lk - Lq if query_start is None else max(-Lq, min(query_start, Lk))
    chunk = min(chunk, max(Lk, 1))
    groups, Lp = pk[0][:2] if pk is not None else (0, 0)
    copied = [(name, shape) for name, (shape, _, _, strides) in zip(_NAMES, metas) if not _layout(shape, strides)]
    for name, shape in copied:
        if shape[1] > 1 and shape[2] * shape[3] >= kernels.ATTENTION_MAX_STRIDE:  # not theirs after a copy either
            _fail(f"the heads of a token of {name} have {shape[2] * shape[3]} elements, they must be fewer than {kernels.ATTENTION_MAX_STRIDE}")
    if copied:
        return None, again
    plan = kernels.past_plan(
        dtype, (B, Lq, Lk, H, Hk, D, groups, Lp), [[s if n > 1 else 0 for s, n in zip(m[3][:3], m[0])] for m in metas],
        0 if window is None else min(max(window, chunk), Lk + chunk), min(sinks, Lk), chunk, start,
        query_start is None and key_lengths is not None and Lq < Lk, scale)
    plan.metas = (_vector(key_lengths), _vector(query_start if isinstance(query_start, tuple) else None), _vector(prefix_lengths),
                  (q[0], dtype, device, (Lq * H * D, H * D, D, 1)), (torch.Size((plan.saved,)), torch.float32, device, (1,)), *metas)
    given = [m for m in plan.metas if m]
    plan.given = ([m[0] for m in given], [m[1] for m in given], [device.index] * len(given), [m[3] for m in given])
    return plan, again


def _vector(meta):
    return meta and (meta[0], torch.int32, meta[2], (1,))


def _int32(t: torch.Tensor | None, low: int, high: int) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype is torch.int64:
        t = t.clamp(low, high).to(torch.int32)
    return t.contiguous()


def _attend(tensors, key_lengths, query_start, prefix_lengths, window, sinks, chunk, scale):
    if not all([isinstance(t, torch.Tensor) for t in tensors]):
        _check_tensors(**dict(zip(_NAMES, tensors)))
    if key_lengths is not None and not isinstance(key_lengths, torch.Tensor):
        _check_tensors(key_lengths=key_lengths)
    if prefix_lengths is not None and not isinstance(prefix_lengths, torch.Tensor):
        _check_tensors(prefix_lengths=prefix_lengths)
    if scale is not None:
        scale = kernels.number("scale", scale, _fail)
    start = query_start
    if isinstance(start, torch.Tensor) and start.dim():
        start = _meta(start)
    elif start is not None:
        start, query_start = _whole("query_start", start), None
    call = _plan(tuple([_meta(t) for t in tensors]), _meta(key_lengths), start, _meta(prefix_lengths),
                 None if window is None else _whole("window", window), _whole("sinks", sinks), _whole("chunk", chunk), scale)
    if key_lengths is not None:
        key_lengths = _int32(key_lengths, 0, tensors[1].shape[1])
    if query_start is not None:
        query_start = _int32(query_start, -tensors[0].shape[1], tensors[1].shape[1])
    if prefix_lengths is not None:
        prefix_lengths = _int32(prefix_lengths, 0, tensors[3].shape[1])
    if kernels.wants_grad(tensors):
        return PastAttentionFunction.apply(call, key_lengths, query_start, prefix_lengths, *tensors)
    plan, tensors, pointers = _lay_out(call, tensors)
    return kernels.past_attention(plan, tensors, pointers, key_lengths, query_start, prefix_lengths)[0]


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, window: int | None = None, sinks: int = 0,
                     chunk: int = 1, key_lengths: torch.Tensor | None = None, query_start: torch.Tensor | int | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """softmax(scale q kᵀ) v per head over the keys that a token sees, [B, Lq, H, D] contiguous in q's dtype.

    q [B, Lq, H, D], k and v [B, Lk, Hk, D], bfloat16 or float32, D a multiple of 8 up to 128. window: how many keys up
    to the end of its own chunk a token sees (at least chunk; None: all before it too). sinks: the first keys that stay visible.
    chunk: tokens that see each other (1: each sees itself and those before it). key_lengths: int32 or int64 [B] on q's device,
    the number of leading keys a sample has (clamped to [0, Lk]). query_start: the position of q's first token, a whole
    number or int32 / int64 [B] on q's device; if not given, the queries are the last Lq of Lk tokens, and with key_lengths and
    Lq < Lk the last Lq of each sample's (a cache). scale > 0, 1 / sqrt(D) if not given."""
    return _attend((q, k, v), key_lengths, query_start, None, window, sinks, chunk, scale)


def prefix_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, prefix_k: torch.Tensor, prefix_v: torch.Tensor, *,
                     window: int | None = None, chunk: int = 1, key_lengths: torch.Tensor | None = None,
                     prefix_lengths: torch.Tensor | None = None, query_start: torch.Tensor | int | None = None,
                     scale: float | None = None) -> torch.Tensor:
    """window_attention of samples that continue a common prefix: every token sees all keys of its prefix as well.

    prefix_k and prefix_v: [Lp, Hk, D] for all samples, or [groups, Lp, Hk, D], each for B / groups samples in a row.
    prefix_lengths: int32 or int64 [groups] on q's device, the leading keys a prefix has (clamped to [0, Lp]). k and v hold the
    samples' own keys; positions, window, chunk and key_lengths count these alone."""
    _check_tensors(prefix_k=prefix_k, prefix_v=prefix_v)
    if prefix_k.dim() == 3 and prefix_v.dim() == 3:
        prefix_k, prefix_v = prefix_k.unsqueeze(0), prefix_v.unsqueeze(0)
    return _attend((q, k, v, prefix_k, prefix_v), key_lengths, query_start, prefix_lengths, window, 0, chunk, scale)

"""The operators between a DiT block's linears in 64 bits on the CPU, straight from their formulas, for
the tests of the kernels. Every function returns what it says as float64 tensors."""
from __future__ import annotations

import math

import torch


def f64(t):
    return None if t is None else t.detach().double().cpu()


def half_step(dtype):
    """The most that one rounding to `dtype` moves a value, relative to it."""
    return torch.finfo(dtype).eps / 2


def rotary(x, w, positions, axis_dims, pairing, theta, eps, g=None):
    """(y, dx, dw, size) of the normed and rotated x [B, L, H, D]; `size` [B, L, 1, 1] bounds the values that the
    rotation adds (the largest normed value of the token). dx and dw are None without g, dw without w."""
    x, w, g, positions = f64(x), f64(w), f64(g), f64(positions)
    if positions.dim() == 2:
        positions = positions.unsqueeze(0)
    B, L, H, D = x.shape
    phi = torch.empty(positions.shape[0], L, D // 2, dtype=torch.float64)
    p = 0
    for c, d in enumerate(axis_dims):
        for i in range(d // 2):
            phi[..., p] = positions[..., c] * theta ** (-2.0 * i / d)
            p += 1
    cos, sin = torch.cos(phi).unsqueeze(2), torch.sin(phi).unsqueeze(2)

    def turn(v, sin):
        a, b = (v[..., 0::2], v[..., 1::2]) if pairing == "adjacent" else (v[..., :D // 2], v[..., D // 2:])
        out = torch.empty_like(v)
        na, nb = a * cos - b * sin, a * sin + b * cos
        if pairing == "adjacent":
            out[..., 0::2], out[..., 1::2] = na, nb
        else:
            out[..., :D // 2], out[..., D // 2:] = na, nb
        return out

    n = x
    if w is not None:
        per_row = w.numel() == H * D
        dims = (2, 3) if per_row else (3,)
        r = 1 / torch.sqrt(x.square().mean(dim=dims, keepdim=True) + eps)
        n = x * r
        wide = w.view(H, D) if per_row else w.view(1, D)
    y = turn(n if w is None else n * wide, sin)
    size = (n if w is None else n * wide).abs().amax(dim=(2, 3), keepdim=True) if L and B else None
    if g is None:
        return y, None, None, size
    back = turn(g, -sin)
    if w is None:
        return y, back, None, size
    dw = (back * n).sum(dim=(0, 1))
    h = back * wide
    dx = r * (h - n * (h * n).mean(dim=dims, keepdim=True))
    return y, dx, dw.reshape(-1) if per_row else dw.sum(dim=0), size


def joint(x, y, gate, scale, shift, post_w, *, norm, post, unit_offset, alpha, eps, gx=None, go=None):
    """(x1, out, grads, sizes): grads a dict of the operands' gradients (vectors per sample, [B, W]); sizes, under
    the same names and "x1" / "out", what each value is made of: the magnitudes its float32 errors are relative to."""
    x, y, gate, scale, shift, post_w, gx, go = map(f64, (x, y, gate, scale, shift, post_w, gx, go))
    W = x.shape[2]
    row = lambda v: None if v is None else v.reshape(-1, 1, W)  # noqa: E731

    def normed(u, kind):
        c = u - u.mean(-1, keepdim=True) if kind == "layer" else u
        r = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + eps)
        return c * r, r

    def back(h, n, r, kind):
        d = h - n * (h * n).mean(-1, keepdim=True)
        return r * (d - h.mean(-1, keepdim=True) if kind == "layer" else d)

    one = torch.ones(1, 1, W, dtype=torch.float64)
    gt = one if gate is None else row(gate)
    pw = one if post_w is None else row(post_w)
    p = y
    if post is not None:
        pn, pr = normed(y, post)
        p = pn * pw
    u = alpha * x + gt * p
    n, r = normed(u, norm)
    m = one if scale is None else row(scale) + (1 if unit_offset else 0)
    out = n * m + (0 if shift is None else row(shift))
    most = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
    sizes = {"x1": (alpha * x).abs() + gt.abs() * most(p) * (1 if post is None else 1 + most(y) * pr)}
    su = most(sizes["x1"]) * r  # of û: the row's largest value over sigma
    sizes["out"] = su * m.abs() + (out - n * m).abs()
    if gx is None and go is None:
        return u, out, None, sizes
    gx, go = (torch.zeros_like(x) if t is None else t for t in (gx, go))
    du = gx + back(go * m, n, r, norm)
    dp = du * gt
    dy = dp if post is None else back(dp * pw, pn, pr, post)
    grads = {"x": alpha * du, "y": dy}
    sdu = gx.abs() + r * most(go * m) * (2 + su) * su.clamp_min(1)
    sdp = sdu * gt.abs()
    sizes["x"] = abs(alpha) * sdu
    sizes["y"] = sdp if post is None else pr * most(sdp * pw) * (2 + most(pn)) * (1 + most(y) * pr)
    sp = most(p) * (1 if post is None else 1 + most(y) * pr)
    for name, t, size in (("gate", du * p, sdu * sp), ("scale", go * n, go.abs() * su), ("shift", go, go.abs()),
                          ("post", dp * pn if post is not None else None, sdp * (1 + most(y) * (pr if post is not None else 1)))):
        if t is not None:
            grads[name], sizes[name] = t.sum(1), size.sum(1)
    return u, out, grads, sizes


def attention(q, k, v, *, live=None, scale=None, do=None):
    """(out, dq, dk, dv, parts) of softmax(scale q k^T) v over the live keys ([B, Lk] bool, None: all); a
    query without keys gets zeros. parts: what the tolerances of the kernels' roundings need, a dict."""
    q, k, v, do = map(f64, (q, k, v, do))
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = H // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    live = torch.ones(B, Lk, dtype=torch.bool) if live is None else live.cpu()
    k, v = (torch.where(live[:, :, None, None], t, torch.zeros_like(t)) for t in (k, v))  # whatever lies there
    qh = q.transpose(1, 2)
    kh, vh = (t.transpose(1, 2).repeat_interleave(G, dim=1) for t in (k, v))
    s = torch.matmul(qh, kh.transpose(-1, -2)) * scale
    s = s.masked_fill(~live[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True) if Lk else torch.zeros(B, H, Lq, 1, dtype=torch.float64)
    m = torch.where(m.isinf(), torch.zeros_like(m), m)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.matmul(p, vh)
    parts = {"out": torch.sqrt(torch.matmul(p.square(), vh.square())).transpose(1, 2),
             "out_abs": torch.matmul(p, vh.abs()).transpose(1, 2), "p": p, "s_abs": torch.matmul(qh.abs(), kh.abs().transpose(-1, -2)) * scale}
    if do is None:
        return o.transpose(1, 2), None, None, None, parts
    g = do.transpose(1, 2)
    delta = (g * o).sum(-1, keepdim=True)
    dp = torch.matmul(g, vh.transpose(-1, -2))
    ds = p * (dp - delta) * scale
    fold = lambda t: t.view(B, Hk, G, Lk, D).sum(2).transpose(1, 2)  # noqa: E731
    dq, dk, dv = torch.matmul(ds, kh), torch.matmul(ds.transpose(-1, -2), qh), torch.matmul(p.transpose(-1, -2), g)
    # absolute sums: what errors relative to P, dP and delta can add up to
    dabs = p * (torch.matmul(g.abs(), vh.abs().transpose(-1, -2)) + (g.abs() * torch.matmul(p, vh.abs())).sum(-1, keepdim=True)) * scale
    parts.update(dq=torch.matmul(dabs, kh.abs()).transpose(1, 2), dk=fold(torch.matmul(dabs.transpose(-1, -2), qh.abs())),
                 dv=fold(torch.matmul(p.transpose(-1, -2), g.abs())))
    return o.transpose(1, 2), dq.transpose(1, 2), fold(dk), fold(dv), parts


def finite_difference(f, x, direction, step):
    """(f(x + step d) - f(x - step d)) / (2 step) for a float64 scalar function."""
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)

"""Attention of tokens to their own past in 64 bits on the CPU, straight from its definition, for the tests of the kernels."""
from __future__ import annotations

import math

import torch

from block_reference import f64, half_step


def starts_of(B, Lq, Lk, lengths=None, start=None):
    """(keys, position of the first query) of every sample."""
    n = [Lk] * B if lengths is None else [min(max(int(v), 0), Lk) for v in lengths]
    if start is None:
        return [(k, k - Lq if lengths is not None and Lq < Lk else Lk - Lq) for k in n]
    first = [int(start)] * B if not isinstance(start, torch.Tensor) else [int(v) for v in start]
    return list(zip(n, first))


def seen(Lq, Lk, n, start, window, sinks, chunk):
    """[Lq, Lk] bool, key by key from the definition."""
    p = torch.arange(Lq).view(-1, 1) + start
    j = torch.arange(Lk).view(1, -1)
    end = (torch.div(p, chunk, rounding_mode="floor") + 1) * chunk
    vis = (j < end) & (j < n) & (p >= 0) & (p < n)
    if window is not None:
        vis &= (j >= end - window) | (j < sinks)
    return vis


def attention(q, k, v, pk=None, pv=None, *, lengths=None, start=None, plens=None, window=None, sinks=0, chunk=1, scale=None, do=None):
    """(outs, parts): outs a dict of out and, with do, dq, dk, dv (dpk, dpv); parts, under the same names, the sums of absolute
    values that errors relative to the weights are made of. Tensors that no token sees may hold anything."""
    dtype = q.dtype
    q, k, v, pk, pv, do = map(f64, (q, k, v, pk, pv, do))
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1:3]
    G = H // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    names = ["out"] + (["dq", "dk", "dv"] if do is not None else []) + (["dpk", "dpv"] if do is not None and pk is not None else [])
    like = {"out": q, "dq": q, "dk": k, "dv": v, "dpk": pk, "dpv": pv}
    outs, parts = ({n: torch.zeros_like(like[n]) for n in names} for _ in range(2))
    s_abs = 0.0
    for b, (n, first) in enumerate(starts_of(B, Lq, Lk, lengths, start)):
        vis = seen(Lq, Lk, n, first, window, sinks, chunk)
        rows = vis.any(1).nonzero().flatten()
        if rows.numel() == 0:
            continue
        keys = vis.any(0).nonzero().flatten()
        vis = vis[rows][:, keys]
        m = 0
        if pk is not None:
            g = b * pk.shape[0] // B
            m = pk.shape[1] if plens is None else min(max(int(plens[g]), 0), pk.shape[1])
            vis = torch.cat((torch.ones(rows.numel(), m, dtype=torch.bool), vis), dim=1)
        for h in range(H):
            hk = h // G
            qq, kk, vv = q[b, rows, h], k[b, keys, hk], v[b, keys, hk]
            if m:
                kk, vv = torch.cat((pk[g, :m, hk], kk)), torch.cat((pv[g, :m, hk], vv))
            p = torch.softmax((scale * qq @ kk.T).masked_fill(~vis, -math.inf), dim=1)
            s_abs = max(s_abs, float((scale * qq.abs() @ kk.abs().T).max()))
            o = p @ vv
            outs["out"][b, rows, h] = o
            parts["out"][b, rows, h] = p @ vv.abs()
            if do is None:
                continue
            g_ = do[b, rows, h]
            dp = g_ @ vv.T
            ds = p * (dp - (g_ * o).sum(1, keepdim=True)) * scale
            dabs = p * (g_.abs() @ vv.abs().T + (g_.abs() * (p @ vv.abs())).sum(1, keepdim=True)) * scale
            outs["dq"][b, rows, h], parts["dq"][b, rows, h] = ds @ kk, dabs @ kk.abs()
            gk, gka, gv, gva = ds.T @ qq, dabs.T @ qq.abs(), p.T @ g_, p.T @ g_.abs()
            outs["dk"][b, keys, hk] += gk[m:]
            parts["dk"][b, keys, hk] += gka[m:]
            outs["dv"][b, keys, hk] += gv[m:]
            parts["dv"][b, keys, hk] += gva[m:]
            if m:
                outs["dpk"][g, :m, hk] += gk[:m]
                parts["dpk"][g, :m, hk] += gka[:m]
                outs["dpv"][g, :m, hk] += gv[:m]
                parts["dpv"][g, :m, hk] += gva[:m]
    return outs, parts, s_abs, dtype


def check(got, q, k, v, pk=None, pv=None, *, do=None, **kw):
    """got: a dict of out and the gradients. Tolerances, value by value, with u half a step of the tensors' type.

    e, what an error relative to every weight can be: two times the error of a score (D products and their sum, the scale
    and the base-2 logarithm's fma in float32: (D + 4) 2^-24 of the sum of absolute products), 2^-20 for exp2, the sum's
    chain and the quotient; in bf16 u more, for the weights' (out, dv) or dS's (dq, dk) rounding as an operand. Then
      out:     u |out| + e (sum p |v| + |out|) + n 2^-24 sum p |v|
      dv:      u |dv| + (e + n 2^-24) sum p |do|
      dq, dk:  u |d| + (e + 2^-17 + (n + D) 2^-24) sum p (|do||v| + |do| sum p |v|) |k or q|
    2^-17: delta is formed from out in two bf16 parts. n: the length of the sum. Weights below 2^-126 are lost to the type's
    range: below 2^-96 in all, allowed beside the rest."""
    outs, parts, s_abs, dtype = attention(q, k, v, pk, pv, do=do, **kw)
    u, D = half_step(dtype), q.shape[3]
    e = 2 * (D + 4) * 2 ** -24 * s_abs + 2 ** -20 + (u if dtype is torch.bfloat16 else 0.0)
    keys = k.shape[1] + (pk.shape[1] if pk is not None else 0)
    rows = q.shape[1] * q.shape[2] // k.shape[2] * (q.shape[0] // pk.shape[0] if pk is not None else 1)
    assert set(got) == set(outs)
    for name, want in outs.items():
        have = f64(got[name])
        assert got[name].dtype == dtype and have.shape == want.shape and got[name].is_contiguous(), name
        n = (keys if name in ("out", "dq") else rows) * 2 ** -24
        rel = e + n + (2 ** -17 + D * 2 ** -24 if name in ("dq", "dk", "dpk") else 0.0)
        room = u * want.abs() + rel * (parts[name] + (want.abs() if name == "out" else 0)) + 2 ** -96
        over = ((have - want).abs() - room).nan_to_num(nan=math.inf)
        at = int(over.argmax()) if over.numel() else 0
        assert over.numel() == 0 or float(over.max()) <= 0, \
            (name, int((over > 0).sum()), at, float(have.reshape(-1)[at]), float(want.reshape(-1)[at]), float(over.reshape(-1)[at]))

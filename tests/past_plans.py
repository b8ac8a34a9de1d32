"""Training calls, bf16 and 128 channels, that between them take every way in which dk and dv are cut: 256 or 128 keys per
workgroup (8 or 4 waves of different keys), and rows shared out or not for the blocks of a prefix, those that hold sinks and the
others. The smallest calls that take them."""
from __future__ import annotations

# groups (0: no prefix), samples per group, tokens, prefix, H, Hk, window, sinks, chunk; waves, shares of dq, of the prefix's, the
# sinks' and the other blocks
PLANS = [
    (0, 1, 700, 0, 64, 8, 100, 400, 1, 8, 1, 1, 11, 7),
    (0, 1, 1000, 0, 32, 8, 100, 400, 1, 8, 1, 1, 10, 4),
    (0, 2, 700, 0, 64, 16, 100, 400, 1, 8, 1, 1, 3, 2),
    (0, 4, 1000, 0, 64, 8, 300, 400, 1, 8, 1, 1, 4, 2),
    (0, 1, 1300, 0, 32, 32, 100, 200, 50, 8, 1, 1, 3, 1),
    (0, 3, 1300, 0, 8, 8, 100, 200, 1, 8, 1, 1, 3, 1),
    (0, 3, 500, 0, 64, 1, 300, 0, 50, 8, 1, 1, 1, 42),
    (0, 1, 1700, 0, 32, 8, None, 0, 1, 8, 1, 1, 1, 5),
    (1, 4, 300, 500, 16, 16, 100, 0, 1, 8, 1, 4, 1, 1),
    (2, 3, 300, 500, 64, 16, 100, 0, 1, 8, 1, 3, 1, 1),
    (1, 3, 500, 1500, 8, 2, 100, 0, 1, 8, 2, 16, 1, 4),
    (1, 3, 1300, 1500, 8, 4, None, 0, 1, 8, 2, 6, 1, 2),
    (1, 2, 1000, 500, 64, 16, None, 0, 1, 8, 1, 4, 1, 2),
    (0, 2, 300, 0, 64, 64, 100, 4, 1, 8, 1, 1, 1, 1),
    (1, 1, 300, 500, 64, 64, 100, 0, 1, 8, 1, 1, 1, 1),
    (0, 3, 700, 0, 32, 8, 300, 4, 1, 4, 1, 1, 3, 2),
    (0, 1, 700, 0, 32, 16, 100, 4, 1, 4, 1, 1, 5, 2),
    (0, 3, 1000, 0, 8, 8, 300, 200, 50, 4, 1, 1, 2, 1),
    (0, 1, 1700, 0, 16, 8, None, 0, 1, 4, 1, 1, 1, 3),
    (1, 3, 300, 500, 64, 8, 300, 0, 1, 4, 1, 7, 1, 2),
    (1, 4, 500, 1500, 4, 4, 300, 0, 50, 4, 4, 4, 1, 1),
    (1, 2, 500, 1500, 4, 4, 300, 0, 50, 4, 4, 4, 1, 2),
]


def ceil_div(a, b):
    return -(-a // b)


def workspace_bytes(case):
    """(dq's, dk / dv's) bytes of the backward's workspace when a call is cut as the row says, each with the rows' deltas."""
    groups, each, L, Lp, H, Hk, window, sinks, _, waves, dq, *splits = case
    B, keys = max(groups, 1) * each, 32 * waves
    rows = H // Hk * L
    blocks = ceil_div(L, keys)
    sink = min(ceil_div(sinks, keys), blocks) if window is not None and window < L else 0
    items = (groups * Hk * ceil_div(Lp, keys), B * Hk * sink, B * Hk * (blocks - sink))
    share = waves * 2 * 4 * 4 * 64  # 16-byte vectors: dk and dv of 128 channels, 32 keys per wave
    dkv = sum(n * s * share for n, s in zip(items, splits) if s > 1)
    return [16 * (ceil_div(B * Hk * rows, 4) + n) for n in (dq * B * Hk * ceil_div(rows, 128) * 4096 if dq > 1 else 0, dkv)]

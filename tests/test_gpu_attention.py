"""Attention to an encoder's states against the 64-bit formulas.

Tolerances, value by value. u: half a step of the output's type, once for the output itself. e: what an error
relative to every weight can be: two times the error of a score (D products and their sum, the scale and the
base-2 logarithm's fma in float32: (D + 4) 2^-24 of the sum of absolute products), 2^-20 for exp2, the sum's
chain and the quotient, and, where the weights are rounded to bf16 for the product with v, u more. Then
  out:      u |out| + e (sum p |v| + |out|)                      (numerator and denominator), + n 2^-24 sum p |v|
  dv:       u |dv|  + (e + n 2^-24) sum p |do|
  dq, dk:   u |d|   + (e + u' + D 2^-24 + n 2^-24) sum p (|do||v| + |do| sum p |v|) ...
with u' one more half step for bf16: delta is formed from the rounded output, and e's own half step stands for
dS's rounding. n: the length of the sum (keys or rows), each addition half a float32 step of the absolute sum.
A weight below 2^-126 is lost to the type's range: 2^-126 each, times at most 2^9 terms of 2^8 |q| < 2^6 and
|do| |v| < 2^12: below 2^-96, allowed beside the rest."""
import math

import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def make(B, Lq, Lk, H, Hk, D, dtype, dev, seed, loud=1.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)  # noqa: E731
    return r(B, Lq, H, D, std=loud), r(B, Lk, Hk, D), r(B, Lk, Hk, D), r(B, Lq, H, D)


def live_keys(B, Lk, lengths=None, mask=None):
    live = torch.ones(B, Lk, dtype=torch.bool)
    if lengths is not None:
        live &= torch.arange(Lk) < lengths.cpu().long().view(B, 1)
    if mask is not None:
        live &= mask.cpu().view(-1, Lk)
    return live


def worst(name, over, got, want):
    over = over.nan_to_num(nan=math.inf)
    at = int(over.argmax())
    return name, int((over > 0).sum()), at, float(got.reshape(-1)[at]), float(want.reshape(-1)[at]), float(over.reshape(-1)[at])


def check(q, k, v, out, g=None, grads=None, *, live=None, scale=None):
    D, u = q.shape[3], ref.half_step(q.dtype)
    o, dq, dk, dv, parts = ref.attention(q, k, v, live=live, scale=scale, do=g)
    low = q.dtype is BF
    s_abs = float(parts["s_abs"].max()) if parts["s_abs"].numel() else 0.0
    e = 2 * (D + 4) * 2 ** -24 * s_abs + 2 ** -20 + (u if low else 0.0)
    n = lambda length: length * 2 ** -24  # noqa: E731
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    diff = (ref.f64(out) - o).abs()
    over = diff - (u * o.abs() + e * (parts["out_abs"] + o.abs()) + n(k.shape[1]) * parts["out_abs"] + 2 ** -96)
    assert (over <= 0).all(), worst("out", over, out, o)
    if g is None:
        return
    more = e + (u if low else 0.0) + n(D)
    rows = q.shape[1] * q.shape[2] // k.shape[2]
    for name, got, want, tol in (("dq", grads[0], dq, more + n(k.shape[1])), ("dk", grads[1], dk, more + n(rows)),
                                 ("dv", grads[2], dv, e + n(rows))):
        diff = (ref.f64(got) - want).abs()
        over = diff - (u * want.abs() + tol * parts[name] + 2 ** -96)
        assert got.shape == want.shape and (over <= 0).all(), worst(name, over, got, want)


def run(pkg, q, k, v, g, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = pkg.cross_attention(*leaves, **kw)
    return out.detach(), torch.autograd.grad(out, leaves, [g])


SHAPES = [
    (1, 1, 1, 1, 1, 8),        # one token, one key
    (2, 1, 77, 12, 12, 128),   # one new token per sample
    (1, 5, 300, 6, 2, 128),    # few rows of heads that share keys (15 per key head)
    (2, 16, 33, 24, 8, 64),    # 48 rows per key head
    (2, 33, 130, 3, 1, 40),    # 99 rows, channels that end inside a step
    (3, 65, 64, 2, 2, 72),     # exactly one key tile; one row past two blocks
    (1, 200, 65, 4, 4, 96),    # one key past a tile
    (1, 129, 513, 2, 1, 128),  # one row and one key past whole tiles
    (2, 250, 7, 5, 5, 64),     # fewer keys than a block
]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("keys", ["all", "lengths", "mask", "both"])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(pkg, dev, shape, keys, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, g = make(*shape, dtype, dev, sum(shape))
    gen = torch.Generator().manual_seed(Lk)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32) if keys in ("lengths", "both") else None
    mask = torch.rand(B, Lk, generator=gen) < 0.6 if keys in ("mask", "both") else None
    live = live_keys(B, Lk, lengths, mask)
    kw = dict(key_lengths=None if lengths is None else lengths.to(dev), key_mask=None if mask is None else mask.to(dev))
    out, grads = run(pkg, q, k, v, g, **kw)
    check(q, k, v, out, g, grads, live=live)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("shape", [
    (1, 3, 5000, 4, 2, 128),   # few rows, the keys split over workgroups and joined
    (1, 40, 4099, 2, 2, 64),
    (2, 100, 3000, 1, 1, 128),  # a whole tile of rows, split
    (1, 2500, 70, 2, 1, 128),  # few keys: the rows of dk and dv split
    (1, 1300, 300, 1, 1, 64),
])
def test_split_and_joined(pkg, dev, shape, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, g = make(*shape, dtype, dev, 7)
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(3)) < 0.8
    lengths = torch.tensor([Lk // 3] * B, dtype=torch.int64)  # later splits have no key
    kw = dict(key_lengths=lengths.to(dev), key_mask=mask.to(dev))
    out, grads = run(pkg, q, k, v, g, **kw)
    check(q, k, v, out, g, grads, live=live_keys(B, Lk, lengths, mask))
    full = run(pkg, q, k, v, g)
    check(q, k, v, full[0], g, full[1])
    again = run(pkg, q, k, v, g)
    assert torch.equal(full[0], again[0]) and all(torch.equal(a, b) for a, b in zip(full[1], again[1]))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq", [1, 40, 150])
def test_rows_without_keys_and_garbage_in_masked_places(pkg, dev, Lq, dtype):
    """A sample without any key gives zeros and zero gradients; NaN, infinities and the type's lowest value in
    masked keys and values change nothing; a wholly masked tile between live ones is skipped."""
    B, Lk, H, D = 4, 320, 2, 64
    q, k, v, g = make(B, Lq, Lk, H, H, D, dtype, dev, 11)
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(1)) < 0.5
    mask[0] = False
    mask[1, 64:192] = False
    mask[3] = False
    mask[3, 300] = True  # a single key
    lengths = torch.tensor([Lk, Lk, 0, Lk], dtype=torch.int32)
    live = live_keys(B, Lk, lengths, mask)
    kw = dict(key_lengths=lengths.to(dev), key_mask=mask.to(dev))
    out, grads = run(pkg, q, k, v, g, **kw)
    check(q, k, v, out, g, grads, live=live)
    for t in (out, *grads):
        assert t[0].abs().sum() == 0 and t[2].abs().sum() == 0
    # a single key's weight is P = 2^d, d the rounding of its score's product with the scale. bf16 rounds P to 1: the
    # value itself. float32 returns fl(fl(v P) fl(1 / P)): three roundings of at most 2^-24 each, below 2^-22.
    want = v[3, 300].expand(Lq, H, D)
    assert torch.equal(out[3], want) if dtype is BF else ((out[3] - want).abs() <= 2 ** -22 * want.abs()).all()
    k2, v2 = k.clone(), v.clone()
    dead = ~live.to(dev)
    for bad_k, bad_v in ((math.nan, math.inf), (math.inf, math.nan), (torch.finfo(dtype).min, -math.inf)):
        k2[dead], v2[dead] = bad_k, bad_v
        out2, grads2 = run(pkg, q, k2, v2, g, **kw)
        assert torch.equal(out, out2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_lengths_out_of_range_are_clamped(pkg, dev):
    q, k, v, g = make(3, 9, 40, 2, 2, 64, BF, dev, 5)
    for dt in (torch.int32, torch.int64):
        out, grads = run(pkg, q, k, v, g, key_lengths=torch.tensor([-5, 1000, 17], dtype=dt, device=dev))
        check(q, k, v, out, g, grads, live=live_keys(3, 40, torch.tensor([0, 40, 17])))


def test_shared_mask_scale_and_loud_scores(pkg, dev):
    """One mask for all samples (also as a vector), a given scale, scores far beyond the running maximum's slack,
    rising and falling along the keys."""
    q, k, v, g = make(2, 70, 260, 2, 2, 64, BF, dev, 6, loud=6.0)
    ramp = torch.linspace(0.1, 8.0, 260, device=dev).view(1, 260, 1, 1)
    mask = torch.rand(260, generator=torch.Generator().manual_seed(2)) < 0.7
    for keys in (k * ramp.to(BF), k * ramp.flip(1).to(BF)):
        for m in (mask, mask.view(1, -1)):
            out, grads = run(pkg, q, keys, v, g, key_mask=m.to(dev), scale=0.3)
            check(q, keys, v, out, g, grads, live=live_keys(2, 260, None, mask), scale=0.3)


def test_layouts(pkg, dev):
    """q of one packed [B, L, 3, H, D], k and v slices of a joint [B, L, 2, H, D], head-major storage, misaligned
    storage, token strides past the kernels' limit, an expanded batch, a strided mask, a transposed gradient."""
    H, D = 4, 64
    q = torch.randn(2, 50, 3, H, D, device=dev).to(BF)[:, :, 1]
    kv = torch.randn(2, 45, 2, H, D, device=dev).to(BF)
    k, v = kv[:, :, 0], torch.randn(2, H, 45, D, device=dev).to(BF).transpose(1, 2)
    g = torch.randn(2, H, 50, D, device=dev).to(BF).transpose(1, 2)
    mask = (torch.rand(2, 90, generator=torch.Generator().manual_seed(4)) < 0.5)[:, ::2]
    out, grads = run(pkg, q, k, v, g, key_mask=mask.to(dev))
    check(q, k, v, out, g, grads, live=mask)
    odd = torch.randn(2 * 45 * H * D + 3, device=dev).to(BF)[3:].view(2, 45, H, D)
    one = torch.randn(1, 45, H, D, device=dev).to(BF).expand(2, 45, H, D)
    out, grads = run(pkg, q, odd, one, g)
    check(q, odd, one, out, g, grads)
    wide = torch.randn(3, (1 << 22) + 8, device=dev).to(BF).as_strided((1, 3, H, D), (0, (1 << 22) + 8, D, 1))
    out, grads = run(pkg, wide, wide, wide, torch.ones_like(wide))
    check(wide, wide, wide, out, torch.ones_like(wide), grads)


@pytest.mark.parametrize("shape", [(0, 5, 7), (2, 0, 7), (2, 5, 0)])
def test_empty(pkg, dev, shape):
    B, Lq, Lk = shape
    q, k, v, g = make(B, Lq, Lk, 4, 2, 64, BF, dev, 1)
    out, grads = run(pkg, q, k, v, g)
    assert out.shape == q.shape and [d.shape for d in grads] == [q.shape, k.shape, v.shape]
    for t in (out, *grads):
        assert t.abs().sum() == 0


def test_gradient_against_differences(pkg, dev):
    """The kernel's float32 gradients against differences of the 64-bit forward formula."""
    q, k, v, g = make(2, 9, 21, 4, 2, 32, F, dev, 13)
    lengths = torch.tensor([21, 6], dtype=torch.int32)
    live = live_keys(2, 21, lengths)
    _, grads = run(pkg, q, k, v, g, key_lengths=lengths.to(dev))
    args = [ref.f64(t) for t in (q, k, v)]
    for i in range(3):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()

        def f(x, i=i):
            return float((ref.attention(*(x if j == i else t for j, t in enumerate(args)), live=live)[0] * ref.f64(g)).sum())

        want = ref.finite_difference(f, args[i], d, 1e-5)
        got = ref.f64(grads[i]) * d
        assert abs(float(got.sum()) - want) <= 2 ** -15 * float(got.abs().sum()) + 1e-6


def test_partial_gradients_and_no_grad(pkg, dev):
    q, k, v, g = make(1, 30, 40, 2, 2, 64, BF, dev, 17)
    out, (dq, dk, dv) = run(pkg, q, k, v, g)
    with torch.no_grad():
        assert torch.equal(pkg.cross_attention(q, k, v), out)
    kk = k.detach().requires_grad_(True)
    (only,) = torch.autograd.grad(pkg.cross_attention(q, kk, v), [kk], [g])
    assert torch.equal(only, dk)
    x = q.detach().requires_grad_(True)
    with pytest.raises(RuntimeError):  # the backward itself is not differentiable, and says so
        (d,) = torch.autograd.grad(pkg.cross_attention(x, k, v), [x], [g], create_graph=True)
        d.float().sum().backward()


def test_captured_and_replayed(pkg, dev):
    """Forward and backward with splits in a HIP graph, replayed with other inputs and key lengths."""
    q, k, v, g = make(1, 700, 80, 2, 2, 128, BF, dev, 19)
    few = make(1, 2, 3000, 2, 2, 128, BF, dev, 20)
    lengths = torch.tensor([80], dtype=torch.int32, device=dev)
    for t in (q, k, v):
        t.requires_grad_(True)

    def step():
        out = pkg.cross_attention(q, k, v, key_lengths=lengths)
        return [out.detach(), pkg.cross_attention(*few[:3]), *torch.autograd.grad(out, [q, k, v], [g])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        gen = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for t in (q, k, v, g, *few[:3]):
                t.copy_(torch.randn(t.shape, generator=gen))
            lengths.fill_(20 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_wan_shape(pkg, dev):
    """The Wan-1.3B cross attention at a frame's length against float64 on the GPU, head by head."""
    B, Lq, Lk, H, D = 2, 3120, 512, 12, 128
    q, k, v, g = make(B, Lq, Lk, H, H, D, BF, dev, 23)
    out, grads = run(pkg, q, k, v, g)
    for b, h in ((0, 0), (1, 11)):
        sub = [t[b:b + 1, :, h:h + 1] for t in (q, k, v)]
        check(*sub, out[b:b + 1, :, h:h + 1].contiguous(), g[b:b + 1, :, h:h + 1], [d[b:b + 1, :, h:h + 1] for d in grads])


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("shape", [
    (1, 700, 2100, 16, 16, 72),  # rows of dk and dv split although the keys alone are many workgroups
    (1, 300, 1500, 6, 2, 96),    # keys of dq split, several row tiles per key head
])
def test_backward_split_with_many_workgroups(pkg, dev, shape, dtype):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, g = make(*shape, dtype, dev, 19)
    mask = torch.rand(B, Lk, generator=torch.Generator().manual_seed(4)) < 0.9
    out, grads = run(pkg, q, k, v, g, key_mask=mask.to(dev))
    check(q, k, v, out, g, grads, live=live_keys(B, Lk, None, mask))


def test_one_tensor_as_q_k_and_v(pkg, dev):
    """The gradients of its three uses add up: each rounded once, so is each sum (two additions)."""
    x = make(2, 90, 90, 3, 3, 64, BF, dev, 23)[0]
    g = make(2, 90, 90, 3, 3, 64, BF, dev, 24)[3]
    _, (dq, dk, dv) = run(pkg, x, x, x, g)
    leaf = x.detach().requires_grad_(True)
    got, = torch.autograd.grad(pkg.cross_attention(leaf, leaf, leaf), [leaf], [g])
    parts = [ref.f64(t) for t in (dq, dk, dv)]
    room = 2 * ref.half_step(BF) * sum(p.abs() for p in parts)
    assert ((ref.f64(got) - sum(parts)).abs() <= room * (1 + ref.half_step(BF))).all()


def test_finer_operands_of_small_backwards(pkg, dev):
    """Up to 2^30 products the weights and dS enter their products in two parts: beside float32 sums (2^-18 in all
    here) only the gradients' own rounding is left, and delta's from the rounded out: its half step u relative to
    every |do| |out|. Root mean squares: u / sqrt(3) at most for the rounding, the same for out's."""
    q, k, v, g = make(2, 40, 180, 6, 2, 64, BF, dev, 31)
    _, grads = run(pkg, q, k, v, g)
    o, dq, dk, dv, parts = ref.attention(q, k, v, do=g)
    u = ref.half_step(BF)
    for name, got, want in (("dq", grads[0], dq), ("dk", grads[1], dk), ("dv", grads[2], dv)):
        err = float((ref.f64(got) - want).norm() / want.norm())
        slack = 0 if name == "dv" else 0.5  # delta: a fraction of dP's spread, out being a mean over the keys
        assert err <= u / math.sqrt(3) * (1 + slack), (name, err)


@pytest.mark.parametrize("shape, keys", [
    ((1, 2500, 700, 8, 4, 96), "mask"),
    ((2, 17000, 70, 8, 8, 64), "lengths"),
    ((1, 10001, 100, 9, 3, 120), "mask"),
    ((1, 4100, 600, 9, 9, 64), "lengths"),
])
def test_large_backwards(pkg, dev, shape, keys):
    """Beyond 2^30 products, where the weights and dS enter their products rounded to bf16."""
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, g = make(*shape, BF, dev, 41)
    gen = torch.Generator().manual_seed(8)
    lengths = torch.tensor([Lk - 3, Lk // 2][:B], dtype=torch.int32) if keys == "lengths" else None
    mask = torch.rand(B, Lk, generator=gen) < 0.7 if keys == "mask" else None
    kw = dict(key_lengths=None if lengths is None else lengths.to(dev), key_mask=None if mask is None else mask.to(dev))
    out, grads = run(pkg, q, k, v, g, **kw)
    check(q, k, v, out, g, grads, live=live_keys(B, Lk, lengths, mask))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq, Lk", [(3, 50), (3, 3000), (200, 50)])
def test_very_low_scores_are_scores(pkg, dev, Lq, Lk, dtype):
    """Every score -2^103 (exact in bf16 and float32): all keys weigh the same, and none of them is a masked one.
    The weights are 1 and their sum Lk exact: v's sum is off by Lk additions, the output by its own half step."""
    q, k, v, _ = make(1, Lq, Lk, 2, 2, 32, dtype, dev, 5)
    q, k = torch.full_like(q, 2.0 ** 49), torch.full_like(k, -(2.0 ** 49))
    out = pkg.cross_attention(q, k, v, scale=1.0)
    want = ref.f64(v).mean(1, keepdim=True).expand(out.shape)
    room = ref.half_step(dtype) * want.abs() + (Lk + 4) * 2 ** -24 * ref.f64(v).abs().mean(1, keepdim=True)
    assert ((ref.f64(out) - want).abs() <= room * (1 + 2 ** -7)).all()

"""Scores far from zero: a softmax depends on differences of scores only, and float32 holds those of equal scores
exactly at any magnitude.

Every key here is the same vector and every score the same number, exact in bf16 and float32 (products of small
integers and powers of two, sums without rounding). So the weights are 1 / n for n live keys, whatever the score. Off by:
the weights' exponent is 0 (2^0 = 1), their sum n is exact, 1 / n and its logarithm and exponential add at most
2^-20 relative (e below: the logarithm of up to 2^12 in float32 is off by 2^-21, times ln 2; exp2 and products 2^-23 each).
  out:  u |out| + (e + n 2^-24) mean |v|                      u: half a step of the output's type
  dv:   u |dv| + (e + rows 2^-24) sum |do| / n                every row gives do / n; bf16 above 2^30 products: + u
  dk:   dS = (do·v - mean do·v) / n: D products each, delta also from out rounded to bf16 where a sample has more than 64
        keys (u |do| |out|), dS rounded like P.  dk = sum over the rows dS q scale
  dq:   the same dS times one and the same key: exactly zero in mathematics, held below the same bound times |k|"""
import math

import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32

# q entry, k entry (D of each): the score is D q k at scale 1
SCORES = {"5*2^34": (5 * 2.0 ** 14, 2.0 ** 15), "-5*2^34": (-5 * 2.0 ** 14, 2.0 ** 15), "3*2^28": (3 * 2.0 ** 10, 2.0 ** 13),
          "-3*2^28": (3 * 2.0 ** 10, -2.0 ** 13), "7*2^60": (7 * 2.0 ** 30, 2.0 ** 25), "3*2^9": (3.0, 16.0), "-3*2^9": (-3.0, 16.0)}


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("Lq, Lk, keys", [
    (3, 50, "all"),        # few rows
    (3, 3000, "all"),      # ... the keys split and joined
    (20, 700, "mask"),
    (200, 50, "lengths"),  # many rows, one tile of keys
    (300, 300, "mask"),
    (2100, 70, "all"),     # the rows of dk and dv split
    (130, 2500, "lengths"),  # the keys of the forward and of dq split
])
def test_equal_scores_of_any_size(pkg, dev, Lq, Lk, keys, score, dtype):
    equal_scores(pkg, dev, Lq, Lk, keys, score, dtype, 2, 2, 32)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("score", ["-5*2^34", "3*2^28", "3*2^9"])
@pytest.mark.parametrize("Lq, Lk, keys, H, Hk, D", [
    (2, 40, "all", 4, 2, 128),        # few rows and keys
    (40, 900, "mask", 2, 2, 128),
    (150, 100, "lengths", 3, 1, 128),  # one tile of query rows ends within a head
    (150, 300, "mask", 2, 2, 72),
    (2600, 140, "all", 1, 1, 128),     # ... the rows of dk and dv split
    (90, 60, "lengths", 2, 1, 104),    # at most 64 keys
])
def test_equal_scores_of_wide_heads(pkg, dev, Lq, Lk, keys, H, Hk, D, score, dtype):
    equal_scores(pkg, dev, Lq, Lk, keys, score, dtype, H, Hk, D)


def equal_scores(pkg, dev, Lq, Lk, keys, score, dtype, H, Hk, D):
    B, G = 2, H // Hk
    gen = torch.Generator().manual_seed(Lq + Lk)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    qe, ke = SCORES[score]
    q, k = torch.full((B, Lq, H, D), qe, dtype=dtype), torch.full((B, Lk, Hk, D), ke, dtype=dtype)
    v, g = r(B, Lk, Hk, D), r(B, Lq, H, D)
    live = torch.ones(B, Lk, dtype=torch.bool)
    kw = {}
    if keys == "mask":
        live = torch.rand(B, Lk, generator=gen) < 0.5
        kw["key_mask"] = live.to(dev)
    elif keys == "lengths":
        lengths = torch.tensor([Lk, Lk // 2 + 3], dtype=torch.int32)
        live = torch.arange(Lk) < lengths.view(2, 1)
        kw["key_lengths"] = lengths.to(dev)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = pkg.cross_attention(*leaves, scale=1.0, **kw)
    grads = [ref.f64(t) for t in torch.autograd.grad(out, leaves, [g.to(dev)])]
    want, _, dk, dv, _ = ref.attention(q, k, v, live=live, scale=1.0, do=g)
    u, e = ref.half_step(dtype), 2 ** -20
    n = live.sum(1).view(B, 1, 1, 1)
    on = live.view(B, Lk, 1, 1).double()
    v64, g64 = ref.f64(v) * on, ref.f64(g)
    wide = lambda t: t.repeat_interleave(G, dim=2)  # noqa: E731
    fold = lambda t, dim: t.unflatten(dim, (Hk, G)).sum(dim + 1)  # noqa: E731
    mean = wide(v64.abs().sum(1, keepdim=True) / n)
    assert ((ref.f64(out) - want).abs() <= u * want.abs() + (e + Lk * 2 ** -24) * mean).all()
    share = on * fold(g64.abs().sum(1, keepdim=True), 2) / n  # what dv adds up
    assert ((grads[2] - dv).abs() <= u * dv.abs() + (e + G * Lq * 2 ** -24) * share).all()
    # dS of row i and key j: at most (|do| |v| + |do| mean |v|) / n off by these shares
    off = e + 2 * D * 2 ** -24 + (u if dtype is BF else 0)
    size = (torch.einsum("bqhd,bkhd->bhqk", g64.abs(), wide(v64.abs())) + (g64.abs() * mean).sum(-1).transpose(1, 2).unsqueeze(-1)) / n
    size = size * on.view(B, 1, 1, Lk)
    room_k = fold(size.sum(2), 1).transpose(1, 2).unsqueeze(-1) * abs(qe)
    assert ((grads[1] - dk).abs() <= u * dk.abs() + (off + G * Lq * 2 ** -24) * room_k).all()
    room_q = size.sum(3).transpose(1, 2).unsqueeze(-1) * abs(ke)
    assert (grads[0].abs() <= (off + Lk * 2 ** -24) * room_q * (1 + 2 * u)).all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq, Lk", [(2, 90), (2, 2048), (150, 90), (150, 2048)])
def test_two_levels_of_large_scores(pkg, dev, Lq, Lk, dtype):
    """Scores of 5 * 2^34 at some keys and 2^13 less (one step of float32 there) at the others: those weigh nothing
    (2^-11818), wherever they lie, and the others alike."""
    B, H, D = 1, 2, 32
    gen = torch.Generator().manual_seed(Lk)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k = torch.zeros(B, Lq, H, D, dtype=dtype), torch.zeros(B, Lk, H, D, dtype=dtype)
    q[..., 0], k[..., 0] = 5 * 2.0 ** 17, 2.0 ** 17
    low = torch.rand(Lk, generator=gen) < 0.5
    q[..., 1], k[:, low, :, 1] = 2.0 ** 6, -(2.0 ** 7)
    v, g = r(B, Lk, H, D), r(B, Lq, H, D)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = pkg.cross_attention(*leaves, scale=1.0)
    dv = ref.f64(torch.autograd.grad(out, leaves, [g.to(dev)])[2])
    v64, g64, u, n = ref.f64(v), ref.f64(g), ref.half_step(dtype), int((~low).sum())
    want = v64[:, ~low].mean(1, keepdim=True)
    room = u * want.abs() + (2 ** -20 + Lk * 2 ** -24) * v64[:, ~low].abs().mean(1, keepdim=True)
    assert ((ref.f64(out) - want).abs() <= room).all()
    assert dv[:, low].abs().sum() == 0
    want = g64.sum(1, keepdim=True) / n
    assert ((dv[:, ~low] - want).abs() <= u * want.abs() + (2 ** -20 + Lq * 2 ** -24) * g64.abs().sum(1, keepdim=True) / n).all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq, Lk", [(3, 200), (150, 200)])
def test_large_scores_beside_small_ones(pkg, dev, Lq, Lk, dtype):
    """Queries of every magnitude in one call, growing scores along the keys for one half of them and falling for the
    other: large rows leave the small ones as they are (each against the formula)."""
    B, H, D = 1, 2, 32
    gen = torch.Generator().manual_seed(Lq)
    r = lambda *s: torch.randn(*s, generator=gen).to(dtype)  # noqa: E731
    q, k, v, g = r(B, Lq, H, D), r(B, Lk, H, D), r(B, Lk, H, D), r(B, Lq, H, D)
    loud = torch.arange(Lq) % 3 == 1
    q[:, loud] = 0
    q[:, loud, :, 0] = (torch.where(torch.arange(Lq)[loud] % 2 == 0, 1.0, -1.0) * 2.0 ** 40).to(dtype).view(1, -1, 1)
    k[..., 0] = torch.arange(Lk).view(1, Lk, 1).to(dtype)
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    out = pkg.cross_attention(*leaves, scale=1.0)
    got = ref.f64(out)
    want, _, _, _, parts = ref.attention(q, k, v, scale=1.0)
    u = ref.half_step(dtype)
    low = u if dtype is BF else 0
    # the loud rows choose the keys whose (rounded) number is largest or smallest, exactly
    quiet = ~loud
    s_abs = float(parts["s_abs"][:, :, quiet].max())
    e = 2 * (D + 4) * 2 ** -24 * s_abs + 2 ** -20 + low
    room = u * want.abs() + (e + Lk * 2 ** -24) * (parts["out_abs"] + want.abs())
    assert ((got - want).abs()[:, quiet] <= room[:, quiet]).all()
    room = u * want.abs() + (2 ** -20 + Lk * 2 ** -24) * parts["out_abs"]
    assert ((got - want).abs()[:, loud] <= room[:, loud]).all()


def test_a_scale_whose_base_two_form_overflows_is_refused(pkg, dev):
    q = torch.zeros(1, 1, 1, 8, device=dev)
    with pytest.raises(RuntimeError):
        pkg.cross_attention(q, q, q, scale=3e38)
    assert math.isfinite(float(pkg.cross_attention(q, q, q, scale=2e38).sum()))


@pytest.mark.parametrize("dtype", [BF, F])
def test_far_and_few_in_a_captured_graph(pkg, dev, dtype):
    """One capture replayed with scores near and far from zero and with many, few and no live keys: what the backward measures
    is decided on the device, and every replay equals the eager call."""
    B, Lq, Lk, H, D = 2, 140, 300, 2, 64
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(len(s))).to(dtype).to(dev)  # noqa: E731
    q, k, v, g = r(B, Lq, H, D), r(B, Lk, H, D), r(B, Lk, H, D), r(B, Lq, H, D)
    mask = torch.ones(B, Lk, dtype=torch.bool, device=dev)
    for t in (q, k, v):
        t.requires_grad_(True)

    def step():
        out = pkg.cross_attention(q, k, v, key_mask=mask, scale=1.0)
        return [out.detach(), *torch.autograd.grad(out, [q, k, v], [g])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for turn, (size, keep) in enumerate(((1.0, 0.8), (2.0 ** 30, 0.8), (1.0, 0.02), (2.0 ** 30, 0.02), (1.0, 0.0), (2.0, 0.9))):
        gen = torch.Generator().manual_seed(turn)
        with torch.no_grad():
            for t in (q, k, v, g):
                t.copy_(torch.randn(t.shape, generator=gen))
            q.mul_(size)
            mask.copy_(torch.rand(B, Lk, generator=gen) < keep)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b) and torch.isfinite(a).all()

"""bf16 gradients of queries whose softmax rests on few keys, given as leading keys, as a mask or both: where few values
add up, out's rounding to bf16 (which delta = do . out would carry on) and the weights' (which the forward's sum holds)
do not average away.

Root mean squares: rounding to bf16 moves a value of [2^k, 2^(k+1)) by up to 2^(k-8), uniformly, 2^(k-8) / sqrt(3) in the
mean square: `rounding` adds that up over the tensor that is wanted. The squares of N uniform errors add up to their mean
within 0.9 / sqrt(N) of it (one deviation; six are allowed). Beside it stand float32 sums of up to 2^10 terms and what two bf16 parts
of P and dS leave out: 2^-14 in all."""
import math

import pytest
import torch

import block_reference as ref
from test_gpu_attention import live_keys, make, run

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def rounding(want):
    """The mean square error, summed, of `want` rounded to bf16."""
    return float((2.0 ** (torch.floor(torch.log2(want[want != 0].abs())) - 8)).square().sum()) / 3


def only_rounded(q, k, v, g, grads, live):
    """The gradients are the formula's, rounded once."""
    _, dq, dk, dv, _ = ref.attention(q, k, v, live=live, do=g)
    found = {}
    for name, got, want in (("dq", grads[0], dq), ("dk", grads[1], dk), ("dv", grads[2], dv)):
        off, norm = float((ref.f64(got) - want).square().sum()), float(want.square().sum())
        most = rounding(want) * (1 + 6 * 0.9 / math.sqrt(int((want != 0).sum())))
        found[name] = (math.sqrt(off / norm), math.sqrt(most / norm) + 2 ** -14)
    assert all(off <= most for off, most in found.values()), found


@pytest.mark.parametrize("how", ["lengths", "mask", "both", "one mask for all"])
@pytest.mark.parametrize("Lq, Lk, H, Hk, D, n", [
    (200, 512, 4, 4, 128, 5),
    (200, 512, 4, 2, 64, 2),
    (3, 700, 6, 2, 128, 3),
    (60, 900, 8, 8, 72, 30),
    (100, 1000, 8, 8, 128, 64),   # as many as are counted, dq's keys split
    (40, 20000, 2, 2, 128, 17),   # far apart, many splits
    (150, 64, 8, 8, 64, 4),       # one tile
])
def test_few_live_keys(pkg, dev, Lq, Lk, H, Hk, D, n, how):
    """The same error whichever way the same number of keys is given, and however many dead ones lie between them."""
    B = 2
    q, k, v, g = make(B, Lq, Lk, H, Hk, D, BF, dev, Lq + Lk + n)
    gen = torch.Generator().manual_seed(n)
    lengths = mask = None
    if how == "lengths":
        lengths = torch.full((B,), n, dtype=torch.int32)
    else:
        rows = 1 if how == "one mask for all" else B
        mask = torch.zeros(rows, Lk, dtype=torch.bool)
        for b in range(rows):
            mask[b, torch.randperm(Lk - (how == "both"), generator=gen)[:n]] = True
        if how == "both":
            lengths = torch.full((B,), Lk - 1, dtype=torch.int32)
            mask[:, Lk - 1] = True  # behind the length
    kw = dict(key_lengths=None if lengths is None else lengths.to(dev), key_mask=None if mask is None else mask.to(dev))
    _, grads = run(pkg, q, k, v, g, **kw)
    only_rounded(q, k, v, g, grads, live_keys(B, Lk, lengths, mask))


def test_live_keys_at_the_border_of_the_count(pkg, dev):
    """63, 64 and 65 live keys and none, in one batch, under masks, against the formula value by value."""
    from test_gpu_attention import check

    B, Lq, Lk = 4, 70, 700
    q, k, v, g = make(B, Lq, Lk, 2, 2, 64, BF, dev, 3)
    mask = torch.zeros(B, Lk, dtype=torch.bool)
    for b, n in enumerate((63, 64, 65, 0)):
        mask[b, torch.randperm(Lk, generator=torch.Generator().manual_seed(b))[:n]] = True
    out, grads = run(pkg, q, k, v, g, key_mask=mask.to(dev))
    check(q, k, v, out, g, grads, live=mask)
    for t in (out, *grads):
        assert t[3].abs().sum() == 0


@pytest.mark.parametrize("Lq, Lk, Hk", [
    (1, 100, 16),   # few rows
    (1, 3000, 4),   # ... that share keys, split
    (40, 200, 16),
    (70, 100, 16),  # many rows
    (70, 1500, 16),  # ... split
])
def test_weights_add_up_to_one(pkg, dev, Lq, Lk, Hk):
    """Among many keys too the weights may rest on a few: scores of a spread of 8, and the weights' own rounding (bf16, for
    their product with v) must not be in the sum that the backward divides by. Only one row of each head has an upstream
    gradient, so that the sum over the keys of <dv_j, do> / <do, do> is the sum of that row's weights, each dv_j = P_j do
    rounded to bf16. Those roundings are no noise to be averaged: do is bf16 itself, and where one P is within 2^-9 of 1 every
    channel of P do rounds to do, all off to one side. So they are computed: weights off by a factor of 1 -+ 2^-14 (the
    float32 scores and sums) give sums between those of P do (1 -+ 2^-14), each rounded."""
    B, H, D = 4, 16, 128
    q, k, v, g = make(B, Lq, Lk, H, Hk, D, BF, dev, 17, loud=8.0)
    g[:, :Lq // 2] = 0
    g[:, Lq // 2 + 1:] = 0
    if Hk < H:
        g[:, :, torch.arange(H) % (H // Hk) != 0] = 0  # one row for every key head
    _, (_, _, dv) = run(pkg, q, k, v, g)
    do = ref.f64(g)[:, Lq // 2, ::H // Hk]  # [B, Hk, D]
    exact = ref.attention(q, k, v, do=g)[3]  # [B, Lk, Hk, D]
    total = lambda t: (ref.f64(t) * do.unsqueeze(1)).sum((1, 3)) / do.square().sum(-1) - 1  # noqa: E731
    low, want, high = (total((exact * (1 + e)).to(BF)) for e in (-(2.0 ** -14), 0.0, 2.0 ** -14))
    off, room = total(dv) - want, torch.maximum(high - want, want - low)
    rms = lambda t: float(t.square().mean().sqrt())  # noqa: E731
    assert rms(off) <= rms(room), (rms(off), rms(room), float(off.abs().max()))


@pytest.mark.parametrize("B, Lq, Lk, H, Hk, D", [
    (6, 512, 512, 8, 8, 128),
    (40, 300, 700, 4, 2, 96),
    (70, 2000, 130, 1, 1, 64),
])
def test_a_samples_gradients_do_not_depend_on_its_batch(pkg, dev, B, Lq, Lk, H, Hk, D):
    """The first sample alone (below 2^30 products of scores and channels) and among others (beyond in all): as
    exact as before. Both are the same values but for the order of float32 sums, so that their errors, squared and added up,
    agree as closely as the errors of N values that are rounded alike."""
    q, k, v, g = make(B, Lq, Lk, H, Hk, D, BF, dev, 29)
    assert H * Lq * Lk * D <= 2 ** 30 < B * H * Lq * Lk * D
    one = [t[:1] for t in (q, k, v, g)]
    _, alone = run(pkg, *one)
    _, among = run(pkg, q, k, v, g)
    wanted = ref.attention(*one[:3], do=one[3])[1:4]
    for name, a, b, want in zip(("dq", "dk", "dv"), alone, among, wanted):
        x, y = (float((ref.f64(t[:1]) - want).norm() / want.norm()) for t in (a, b))
        assert abs(x - y) <= x * 6 * 0.9 / math.sqrt(want.numel()), (name, x, y)


@pytest.mark.parametrize("Lk", [65, 79, 80, 81, 1023, 1025, 4097, 9001])
@pytest.mark.parametrize("n", [1, 20, 64])
def test_few_keys_of_masks_at_any_address(pkg, dev, Lk, n):
    """Rows of a mask that begin at any byte, live keys at both ends, and set bytes behind the row's end and behind the
    sample's length, which do not count: as exact as the same keys by themselves."""
    B, Lq, H, D = 3, 33, 2, 64
    q, k, v, g = make(B, Lq, Lk, H, H, D, BF, dev, Lk + n)
    gen = torch.Generator().manual_seed(Lk)
    wide = torch.ones(B, Lk + 5, dtype=torch.bool)
    mask = wide[:, 3:3 + Lk]
    mask[:] = False
    lengths = torch.tensor([Lk, Lk - 1, Lk], dtype=torch.int32)
    for b in range(B):
        end = int(lengths[b])
        mask[b, torch.randperm(end - 1, generator=gen)[:n - 1]] = True
        mask[b, end - 1] = True
        mask[b, end:] = True
    kw = dict(key_lengths=lengths.to(dev), key_mask=wide.to(dev)[:, 3:3 + Lk])
    assert kw["key_mask"].stride(0) == Lk + 5
    _, grads = run(pkg, q, k, v, g, **kw)
    live = live_keys(B, Lk, lengths, mask)
    assert live.sum(1).tolist() == [n] * B
    if n > 1:
        only_rounded(q, k, v, g, grads, live)
    else:  # a lone key: dq and dk are zero in mathematics, and dv the sum of do with weights off by 2^-18 at most (the logarithm's
        # rounding, scores below 2^6, and the sum of 33 rows)
        want, g64 = ref.attention(q, k, v, live=live, do=g)[3], ref.f64(g)
        room = ref.half_step(BF) * want.abs() + 2 ** -18 * g64.abs().sum(1, keepdim=True)
        assert ((ref.f64(grads[2]) - want).abs() <= room).all()
    for d in grads[1:]:
        assert d[~live.to(dev)].abs().sum() == 0

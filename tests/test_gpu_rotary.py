"""Rotary positions with several axes, with and without the q / k norms, against the 64-bit formulas.

Tolerances. A result is rounded once to its type (half a step of the value). Before that, in float32: the
cosine and sine are off by at most 2^-23.3 (the reduced turn's rounding, half of 2^-25 times 2 pi) plus 2 ulp of
sincospi (2^-22) < 2^-21.2; the products and the sum add 3 half steps; a norm's 1 / sigma is off by at most half
of (16 values + 1 unit + 6 + 4 additions + mean, root, quotient) half steps, about 15 of 2^-24, and two products:
together below 2^-19.5 of the token's largest normed value for each of the pair's two members, 2^-18.5 in all.
Gradients go through as many steps once more: 2^-17 of the sizes they are made of. A weight's gradient sums at
most 2^15 rows in chains of at most 128 + 4 + 512 / 16 + 16 < 256 additions, each half a step of the sum of
absolute values: 2^-16 of that sum, with 2^-17 of every term before: 2^-15."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu


def make(B, L, H, Hk, D, axes, dtype, norm, seed, dev, fractional=False, far=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).to(dev)  # noqa: E731
    q, k, gq, gk = r(B, L, H, D), r(B, L, Hk, D), r(B, L, H, D), r(B, L, Hk, D)
    pos = torch.randint(0, 200, (B, L, axes), generator=g, dtype=torch.int32) + far
    if fractional:
        pos = pos.float() * 0.37 - 3.3
    ws = [None, None]
    if norm != "none":
        ws = [(1 + 0.2 * torch.randn(h * D if norm == "row" else D, generator=g)).to(dtype).to(dev) for h in (H, Hk)]
    return q, k, gq, gk, pos.to(dev), ws


def check(x, w, pos, axis_dims, pairing, y, g=None, dx=None, dw=None, theta=10000.0, eps=1e-6):
    ry, rdx, rdw, size = ref.rotary(x, w, pos, axis_dims, pairing, theta, eps, g)
    u = ref.half_step(x.dtype)
    assert ((ref.f64(y) - ry).abs() <= u * ry.abs() + 2 ** -18.5 * size).all()
    if g is None:
        return
    xd, gd = ref.f64(x), ref.f64(g)
    if w is None:
        bound = gd.abs().amax(dim=(2, 3), keepdim=True)
    else:
        per_row = w.numel() == x.shape[2] * x.shape[3]
        dims = (2, 3) if per_row else (3,)
        r = 1 / torch.sqrt(xd.square().mean(dim=dims, keepdim=True) + eps)
        h = gd.abs().amax(dim=(2, 3), keepdim=True) * ref.f64(w).abs().max() * 2 ** 0.5
        bound = r * h * (1 + (xd * r).abs())
    assert ((ref.f64(dx) - rdx).abs() <= u * rdx.abs() + 2 ** -17 * bound).all()
    if w is not None:
        n = xd * r
        pair = gd.abs() + (gd.abs().view(*gd.shape[:3], -1, 2).flip(-1).flatten(3) if pairing == "adjacent"
                           else gd.abs().roll(gd.shape[3] // 2, 3))
        terms = (pair * n.abs()).sum(dim=(0, 1))
        terms = terms.reshape(-1) if per_row else terms.sum(0)
        assert ((ref.f64(dw) - rdw).abs() <= ref.half_step(w.dtype) * rdw.abs() + 2 ** -15 * terms).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", ["none", "head", "row"])
@pytest.mark.parametrize("pairing", ["adjacent", "halves"])
@pytest.mark.parametrize("shape", [
    (1, 1, 1, 1, 16, (16,)),              # one token of the smallest head
    (2, 7, 12, 12, 128, (44, 42, 42)),    # Wan's heads and axes
    (1, 33, 8, 1, 64, (32, 32)),          # key heads shared
    (3, 5, 5, 5, 96, (32, 32, 32)),       # heads of six units: sums across lanes
    (2, 9, 40, 8, 128, (44, 42, 42)),     # several waves to a row
    (1, 6, 31, 2, 256, (64, 96, 96)),     # the widest heads, 124 pairs past lane 64
    (1, 130, 3, 3, 48, (0, 16, 32)),      # an axis without channels, three units to a head
])
def test_against_the_formula(pkg, dev, shape, pairing, norm, dtype):
    B, L, H, Hk, D, axes = shape
    q, k, gq, gk, pos, ws = make(B, L, H, Hk, D, len(axes), dtype, norm, sum(shape[:5]), dev)
    leaves = [t.requires_grad_(True) for t in (q, k, *(w for w in ws if w is not None))]
    yq, yk = pkg.rotary_axes_qk(q, k, pos, axes, pairing=pairing, q_weight=ws[0], k_weight=ws[1])
    assert yq.dtype == dtype and yq.shape == q.shape and yk.shape == k.shape and yq.is_contiguous()
    grads = torch.autograd.grad([yq, yk], leaves, [gq, gk])
    dw = grads[2:] if norm != "none" else (None, None)
    check(q, ws[0], pos, axes, pairing, yq, gq, grads[0], dw[0])
    check(k, ws[1], pos, axes, pairing, yk, gk, grads[1], dw[1])


@pytest.mark.parametrize("kind", ["fractional", "far", "int64"])
def test_positions(pkg, dev, kind):
    """Fractional positions, places far out (where 32-bit angles would be off by whole turns), 64-bit integers."""
    axes = (44, 42, 42)
    q, _, g, _, pos, _ = make(2, 19, 4, 4, 128, 3, torch.float32, "none", 5, dev, fractional=kind == "fractional",
                              far=(1 << 24) + 1 if kind != "fractional" else 0)
    if kind == "int64":
        pos = pos.long() + (1 << 26)
    q.requires_grad_(True)
    y = pkg.rotary_axes(q, pos, axes)
    (dq,) = torch.autograd.grad(y, [q], [g])
    check(q, None, pos, axes, "adjacent", y, g, dq)


def test_long_rows_and_weight_sums(pkg, dev):
    """Many tokens: several workgroups' partial rows, a batch that ends inside a workgroup's tokens."""
    axes = (44, 42, 42)
    q, k, gq, gk, pos, ws = make(3, 2111, 12, 12, 128, 3, torch.bfloat16, "row", 6, dev)
    for t in (q, k, *ws):
        t.requires_grad_(True)
    yq, yk = pkg.rotary_axes_qk(q, k, pos, axes, q_weight=ws[0], k_weight=ws[1])
    dq, dk, dqw, dkw = torch.autograd.grad([yq, yk], [q, k, *ws], [gq, gk])
    check(q, ws[0], pos, axes, "adjacent", yq, gq, dq, dqw)
    check(k, ws[1], pos, axes, "adjacent", yk, gk, dk, dkw)
    again = torch.autograd.grad(pkg.rotary_axes_qk(q, k, pos, axes, q_weight=ws[0], k_weight=ws[1]), [q, k, *ws], [gq, gk])
    for a, b in zip((dq, dk, dqw, dkw), again):
        assert torch.equal(a, b)  # the sums' order is fixed


def test_grid_and_padding(pkg, dev):
    """Wan's grids in a padded batch: tokens behind a sample's grid come back bit for bit."""
    pos = pkg.grid_positions([[2, 3, 4], [1, 5, 2]], 30, dev)
    assert pos.shape == (2, 30, 3) and pos[0, 23].tolist() == [1, 2, 3] and pos[1, 10:].abs().sum() == 0
    x = torch.randn(2, 30, 4, 64, device=dev).bfloat16()
    y = pkg.rotary_axes(x, pos, (24, 20, 20))
    check(x, None, pos, (24, 20, 20), "adjacent", y)
    assert torch.equal(y[0, 24:], x[0, 24:]) and torch.equal(y[1, 10:], x[1, 10:])
    later = pkg.grid_positions([[1, 2, 2]], 4, dev, start=(7, 0, 0))
    assert later[0, :, 0].tolist() == [7] * 4


def test_layouts(pkg, dev):
    """Slices of one packed [B, L, 3, H, D], transposed heads, misaligned storage, an expanded batch, one token
    dimension of any stride, and a transposed upstream gradient."""
    axes = (32, 32)
    packed = torch.randn(2, 11, 3, 4, 64, device=dev).bfloat16()
    pos = torch.randint(0, 50, (11, 2), device=dev, dtype=torch.int32)
    w = torch.randn(64, device=dev)
    views = [packed[:, :, 0], torch.randn(2, 4, 11, 64, device=dev).bfloat16().transpose(1, 2),
             torch.randn(2 * 11 * 4 * 64 + 3, device=dev).bfloat16()[3:].view(2, 11, 4, 64),
             torch.randn(1, 11, 4, 64, device=dev).bfloat16().expand(2, 11, 4, 64)]
    for x in views:
        x = x.detach().requires_grad_(True)
        y = pkg.rotary_axes(x, pos, axes, weight=w)
        g = torch.randn(2, 4, 11, 64, device=dev).bfloat16().transpose(1, 2)
        (dx,) = torch.autograd.grad(y, [x], [g])
        ry, rdx, _, _ = ref.rotary(x, w, pos, axes, "adjacent", 10000.0, 1e-6, g)
        check(x, w, pos, axes, "adjacent", y)
        assert (ref.f64(dx) - rdx).norm() <= 2 ** -8 * rdx.norm()


def test_empty_and_partial_gradients(pkg, dev):
    axes = (32, 32)
    pos = torch.zeros(0, 2, dtype=torch.int32, device=dev)
    x = torch.randn(2, 0, 4, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = pkg.rotary_axes(x, pos, axes, weight=w)
    dx, dw = torch.autograd.grad(y, [x, w], [torch.zeros_like(y)])
    assert y.shape == x.shape and dx.shape == x.shape and dw.abs().sum() == 0
    # only k's gradient, only a weight's
    q, k, gq, gk, pos, ws = make(2, 9, 4, 4, 64, 2, torch.float32, "head", 3, dev)
    k.requires_grad_(True), ws[0].requires_grad_(True)
    yq, yk = pkg.rotary_axes_qk(q, k, pos, axes, q_weight=ws[0], k_weight=ws[1])
    dk, dqw = torch.autograd.grad([yq, yk], [k, ws[0]], [gq, gk])
    check(k, ws[1], pos, axes, "adjacent", yk, gk, dk, ref.rotary(k, ws[1], pos, axes, "adjacent", 1e4, 1e-6, gk)[2])
    (only,) = torch.autograd.grad(pkg.rotary_axes_qk(q, k, pos, axes, q_weight=ws[0], k_weight=ws[1])[1], [k], [gk])
    assert torch.equal(only, dk) and dqw.shape == (64,)


def test_gradient_against_differences(pkg, dev):
    """The kernel's gradient of a float32 pass against differences of the 64-bit forward formula."""
    axes = (20, 20, 24)
    q, _, g, _, pos, ws = make(1, 5, 3, 3, 64, 3, torch.float32, "row", 9, dev)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(pkg.rotary_axes(q, pos, axes, weight=ws[0]), [q], [g])
    f = lambda x: float((ref.rotary(x, ws[0], pos, axes, "adjacent", 1e4, 1e-6)[0] * ref.f64(g)).sum())  # noqa: E731
    for seed in range(3):
        d = torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)).double()
        want = ref.finite_difference(f, ref.f64(q), d, 1e-5)
        # the difference quotient itself is good to about 1e-9; the gradient to 2^-17 of its terms
        assert abs(float((ref.f64(dq) * d).sum()) - want) <= 2 ** -17 * float((ref.f64(dq).abs() * d.abs()).sum()) + 1e-6


def test_captured_and_replayed(pkg, dev):
    """Forward and backward in a HIP graph, replayed with other inputs, equal to the eager pass."""
    axes = (44, 42, 42)
    q, k, gq, gk, pos, ws = make(1, 300, 4, 4, 128, 3, torch.bfloat16, "row", 11, dev)
    for t in (q, k, *ws):
        t.requires_grad_(True)

    def step():
        y = pkg.rotary_axes_qk(q, k, pos, axes, q_weight=ws[0], k_weight=ws[1])
        return [*(t.detach() for t in y), *torch.autograd.grad(y, [q, k, *ws], [gq, gk])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(4):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            for t in (q, k, gq, gk):
                t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)

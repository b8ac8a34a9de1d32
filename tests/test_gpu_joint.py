"""The joint of two sublayers (norm after, gate, residual, norm before) against the 64-bit formulas.

Tolerances. Every output is rounded once to its type: half a step of the value. Before that, in float32, a row's
sums are at most 3 * 8 values per lane, 6 butterfly steps and 8 waves: 38 additions, half a step (2^-24) of the row's
largest value each; the mean, variance, root, quotient and products add fewer than 20 more: below 2^-18 of the
sizes that the values are made of (the row's largest value over sigma, and so on: the reference's `sizes`). An
output passes at most two norms (2^-17); a gradient passes them once more in the other direction, four in all: 2^-16.
A vector's gradient sums rows in chains of at most 4096 / 4 per stream, 8 streams, 512 / 16 + 16 partial
rows: at the sizes here at most 32 + 8 + 48 < 256 additions, 2^-16 of the terms, whose own errors are 2^-16: 2^-15."""
import pytest
import torch

import block_reference as ref

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def make(B, T, W, stream, dt, dev, seed, *, gate="sample", affine="sample", post=False, vec=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, dtype=F, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)  # noqa: E731
    vec = vec or (F if stream is F else dt)
    shape = {"sample": (B, W), "shared": (W,), "row": (B, 1, W), "one": (1, W)}
    d = dict(x=r(B, T, W, dtype=stream, std=2.0) + 0.5, y=r(B, T, W, dtype=dt),
             gate=None if gate is None else r(*shape[gate], dtype=vec),
             scale=None if affine is None else r(*shape[affine], dtype=vec, std=0.3),
             shift=None if affine is None else r(*shape[affine], dtype=vec),
             post_weight=(1 + r(W, std=0.2)).to(vec) if post else None,
             gx=r(B, T, W, dtype=stream), go=r(B, T, W, dtype=dt))
    return d


def run(pkg, d, **cfg):
    names = [n for n in ("x", "y", "gate", "scale", "shift", "post_weight") if d[n] is not None]
    leaves = [d[n].detach().requires_grad_(True) for n in names]
    a = dict(zip(names, leaves))
    outs = pkg.gated_residual_norm(a["x"], a["y"], a.get("gate"), a.get("scale"), a.get("shift"),
                                   post_weight=a.get("post_weight"), **cfg)
    return [t.detach() for t in outs], dict(zip(names, torch.autograd.grad(outs, leaves, [d["gx"], d["go"]])))


def check(d, outs, grads, norm="layer", post_norm=None, unit_offset=True, residual_scale=1.0, eps=1e-6):
    u, out, want, sizes = ref.joint(d["x"], d["y"], d["gate"], d["scale"], d["shift"], d["post_weight"], norm=norm,
                                    post=post_norm, unit_offset=unit_offset, alpha=residual_scale, eps=eps,
                                    gx=d["gx"], go=d["go"])
    near = lambda a, b, size, tol: ((ref.f64(a) - b).abs() <= ref.half_step(a.dtype) * b.abs() + tol * size).all()  # noqa: E731
    assert outs[0].dtype == d["x"].dtype and outs[1].dtype == d["y"].dtype
    assert near(outs[0], u, sizes["x1"], 2 ** -17), "x1"
    assert near(outs[1], out, sizes["out"], 2 ** -17), "out"
    for name, g in grads.items():
        assert g.shape == d[name].shape and g.dtype == d[name].dtype
        key = "post" if name == "post_weight" else name
        b, size = want[key], sizes[key]
        if name in ("x", "y"):
            assert near(g, b, size, 2 ** -16), name
            continue
        if d[name].numel() == b.shape[1]:  # shared by the samples
            b, size = b.sum(0), size.sum(0)
        assert near(g.reshape(b.shape), b, size, 2 ** -15), name


@pytest.mark.parametrize("types", [(BF, BF), (F, BF), (F, F)])
@pytest.mark.parametrize("norm, post", [("layer", None), ("rms", "rms"), ("layer", "layer"), ("rms", None)])
@pytest.mark.parametrize("shape", [(1, 1, 8), (2, 7, 256), (3, 5, 1536), (2, 9, 2056), (1, 4, 5120), (2, 3, 8192)])
def test_against_the_formula(pkg, dev, shape, norm, post, types):
    d = make(*shape, *types, dev, sum(shape), post=post is not None)
    outs, grads = run(pkg, d, norm=norm, post_norm=post, residual_scale=0.75)
    check(d, outs, grads, norm=norm, post_norm=post, residual_scale=0.75)


@pytest.mark.parametrize("gate", [None, "shared", "row", "one"])
@pytest.mark.parametrize("affine", [None, "shared", "row", "one"])
def test_vectors(pkg, dev, gate, affine):
    """Every shape of the vectors, their gradients summed over the samples where they are shared; norm weights."""
    d = make(3, 13, 264, F, BF, dev, 4, gate=gate, affine=affine, vec=BF)
    outs, grads = run(pkg, d, unit_offset=False)
    check(d, outs, grads, unit_offset=False)


def test_scale_without_shift_and_post_norm_without_weight(pkg, dev):
    d = make(2, 6, 128, BF, BF, dev, 8)
    d["shift"] = None
    outs, grads = run(pkg, d, norm="rms", post_norm="layer")
    check(d, outs, grads, norm="rms", post_norm="layer")


@pytest.mark.parametrize("B, T, W", [(2, 4111, 1536), (600, 3, 64), (5, 700, 2560)])
def test_many_rows(pkg, dev, B, T, W):
    """Many workgroups, chunks that end in the middle, many samples; the vector sums' order is fixed."""
    d = make(B, T, W, F, BF, dev, 21, post=True)
    outs, grads = run(pkg, d, post_norm="rms")
    check(d, outs, grads, post_norm="rms")
    _, again = run(pkg, d, post_norm="rms")
    for k in grads:
        assert torch.equal(grads[k], again[k]), k


def test_wan_chunks_of_the_modulation(pkg, dev):
    """gate, scale and shift as rows of one [B, 6, W] modulation, x a slice of a longer stream, y transposed."""
    d = make(2, 11, 512, F, BF, dev, 31)
    e = torch.randn(2, 6, 512, device=dev)
    d["gate"], d["scale"], d["shift"] = e[:, 2:3], e[:, 4:5], e[:, 3:4]
    long = torch.randn(2, 30, 512, device=dev)
    d["x"] = long[:, 5:16]
    d["y"] = torch.randn(11, 2, 512, device=dev).to(BF).transpose(0, 1)
    outs, grads = run(pkg, d)
    check(d, outs, grads)
    d["y"] = torch.randn(2 * 11 * 512 + 1, device=dev).to(BF)[1:].view(2, 11, 512)  # misaligned storage
    outs, grads = run(pkg, d)
    check(d, outs, grads)


def test_one_output_used_and_frozen_vectors(pkg, dev):
    """Only x1 or only out goes on; the modulation frozen (no sums), only y's gradient wanted."""
    d = make(2, 9, 320, F, BF, dev, 41)
    for keep in (0, 1):
        x, y = d["x"].detach().requires_grad_(True), d["y"].detach().requires_grad_(True)
        outs = pkg.gated_residual_norm(x, y, d["gate"], d["scale"], d["shift"])
        g = (d["gx"], d["go"])[keep]
        dx, dy = torch.autograd.grad(outs[keep], [x, y], [g])
        e = dict(d, **{("go", "gx")[keep]: torch.zeros_like((d["go"], d["gx"])[keep])})
        check(e, [t.detach() for t in outs], {"x": dx, "y": dy})
        outs = pkg.gated_residual_norm(d["x"], y, d["gate"], d["scale"], d["shift"])
        (only,) = torch.autograd.grad(outs[keep], [y], [g])
        assert torch.equal(only, dy)


def test_empty(pkg, dev):
    x = torch.randn(2, 0, 64, device=dev, requires_grad=True)
    y = torch.randn(2, 0, 64, device=dev, requires_grad=True)
    gate, scale = torch.randn(2, 64, device=dev, requires_grad=True), torch.randn(64, device=dev, requires_grad=True)
    outs = pkg.gated_residual_norm(x, y, gate, scale)
    grads = torch.autograd.grad(outs, [x, y, gate, scale], [torch.zeros_like(t) for t in outs])
    assert [g.shape for g in grads] == [x.shape, y.shape, gate.shape, scale.shape]
    assert grads[2].abs().sum() == 0 and grads[3].abs().sum() == 0


def test_gradient_against_differences(pkg, dev):
    """The kernel's float32 gradients against differences of the 64-bit forward formula."""
    d = make(2, 4, 64, F, F, dev, 51, post=True)
    cfg = dict(norm="layer", post="rms", unit_offset=True, alpha=0.5, eps=1e-6)
    _, grads = run(pkg, d, norm="layer", post_norm="rms", residual_scale=0.5)
    names = ("x", "y", "gate", "scale", "shift", "post_weight")

    def total(args):
        u, out, _, _ = ref.joint(*args, **cfg)
        return float((u * ref.f64(d["gx"])).sum() + (out * ref.f64(d["go"])).sum())

    for i, name in enumerate(names):
        direction = torch.randn(d[name].shape, generator=torch.Generator().manual_seed(i)).double()

        def f(v, i=i):
            return total([v if j == i else ref.f64(d[n]) for j, n in enumerate(names)])

        want = ref.finite_difference(f, ref.f64(d[name]), direction, 1e-5)
        got = float((ref.f64(grads[name]) * direction).sum())
        assert abs(got - want) <= 2 ** -15 * float((ref.f64(grads[name]) * direction).abs().sum()) + 1e-6, name


def test_captured_and_replayed(pkg, dev):
    d = make(2, 300, 1536, F, BF, dev, 61)
    for t in d.values():
        if t is not None and t is not d["gx"] and t is not d["go"]:
            t.requires_grad_(True)
    leaves = [d[n] for n in ("x", "y", "gate", "scale", "shift")]

    def step():
        outs = pkg.gated_residual_norm(*leaves)
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, leaves, [d["gx"], d["go"]])]

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
            for n in ("x", "y", "gx", "go"):
                d[n].copy_(torch.randn(d[n].shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("types", [(BF, BF), (F, BF), (F, F)])
@pytest.mark.parametrize("W", [1032, 1544, 2048, 4104, 7168])
def test_widths_between_the_tiles(pkg, dev, W, types):
    """Rows whose last wave or last chunk is partly or wholly empty, all gradients, several workgroups per sample."""
    d = make(2, 300, W, *types, dev, W, post=True)
    outs, grads = run(pkg, d, norm="layer", post_norm="layer")
    check(d, outs, grads, norm="layer", post_norm="layer")

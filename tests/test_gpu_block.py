"""The operators of a block in the order a model runs them, with the LoRA linears between them: modulated norm,
q / k / v, q / k norms and rotary positions, self-attention, o, the joint with the affine norm, cross-attention to a
padded text context, the joint with the modulation, ffn, the last joint. Forward and every gradient against float64
torch autograd on the CPU.

Tolerances (relative 2-norms). float32: a pass through the chain is about 25 operators, each within about 1e-6 of its
exact result (sums of up to 512 products, half a step 6e-8 each), forward and backward: 50 of them, 5e-5 if they
all added up. bf16: each of the about 20 tensors between operators, and in the backward the 20 gradients, is rounded
once (2^-8 at most, about 1.7e-3 in the mean square) and the attention's weights and dS once more: the square
root of 60 roundings of 1.7e-3 is 1.3e-2; a gradient passes both: 2.6e-2, allowed 4e-2 for the norms' gain of errors."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
B, GRID, TXT, HEADS, D, FFN, RANK = 2, (3, 4, 5), 13, 4, 32, 256, 8
L, C = 60 + 4, HEADS * D  # four padding tokens behind the grid
AXES = (12, 10, 10)
LINEARS = {"q": (C, C), "k": (C, C), "v": (C, C), "o": (C, C), "cq": (C, C), "ck": (C, C), "cv": (C, C), "co": (C, C),
           "f0": (C, FFN), "f2": (FFN, C)}


def parameters(dtype, dev):
    g = torch.Generator().manual_seed(77)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)  # noqa: E731
    p = {"x": r(B, L, C).float() if dtype is torch.float32 else r(B, L, C), "text": r(B, TXT, C),
         "table": r(1, 6, C, std=0.1).float(), "time": r(B, 6, C, std=0.3).float(),
         "norm3_w": (1 + r(C, std=0.1).float()), "norm3_b": r(C, std=0.1).float()}
    for n in ("qn", "kn", "cqn", "ckn"):
        p[n] = (1 + r(C, std=0.1).float()).to(dtype)
    for n, (i, o) in LINEARS.items():
        p[n + ".w"], p[n + ".b"] = r(o, i, std=i ** -0.5), r(o, std=0.02)
        p[n + ".a"], p[n + ".bb"] = r(RANK, i, std=i ** -0.5), r(o, RANK, std=0.05)
    return p


TRAINED = ["x", "text", "table", "time", "norm3_w", "norm3_b", "qn", "kn", "cqn", "ckn",
           *(f"{n}.{s}" for n in LINEARS for s in ("a", "bb"))]


def through_kernels(pkg, p, lengths, pos):
    x, text = p["x"], p["text"]
    rows, words = pkg.SegmentRouting.from_lengths([B * L], [0]), pkg.SegmentRouting.from_lengths([B * TXT], [0])

    def lin(n, t):
        y = pkg.multi_lora_linear(t.reshape(-1, t.shape[2]), p[n + ".w"], p[n + ".b"], [p[n + ".a"]], [p[n + ".bb"]], [1.0],
                                  words if t.shape[1] == TXT else rows)
        return y.view(t.shape[0], t.shape[1], -1)

    heads = lambda t: t.unflatten(2, (HEADS, D))  # noqa: E731
    e = p["table"] + p["time"]  # [B, 6, C]
    # the block's first norm, as the joint of the block before would leave it
    stream, y = pkg.gated_residual_norm(x, torch.zeros_like(x), None, e[:, 1], e[:, 0])
    q, k = pkg.rotary_axes_qk(heads(lin("q", y)), heads(lin("k", y)), pos, AXES, q_weight=p["qn"], k_weight=p["kn"])
    a = pkg.cross_attention(q, k, heads(lin("v", y)))
    stream, y = pkg.gated_residual_norm(stream, lin("o", a.flatten(2)), e[:, 2], p["norm3_w"], p["norm3_b"], unit_offset=False)
    q, k = heads(lin("cq", y)), heads(lin("ck", text))
    zero = torch.zeros(1, TXT if TXT > L else L, 1, dtype=torch.int32, device=x.device)
    q = pkg.rotary_axes(q, zero[:, :L], (D,), weight=p["cqn"])  # the origin: the norm alone
    k = pkg.rotary_axes(k, zero[:, :TXT], (D,), weight=p["ckn"])
    a = pkg.cross_attention(q, k, heads(lin("cv", text)), key_lengths=lengths)
    stream, y = pkg.gated_residual_norm(stream, lin("co", a.flatten(2)), None, e[:, 4], e[:, 3])
    y = lin("f2", torch.nn.functional.gelu(lin("f0", y), approximate="tanh"))
    return pkg.gated_residual_norm(stream, y, e[:, 5], norm="rms")


def exactly(p, lengths, pos):
    x, text = p["x"], p["text"]

    def lin(n, t):
        return t @ p[n + ".w"].T + p[n + ".b"] + t @ p[n + ".a"].T @ p[n + ".bb"].T

    def layer(t):
        c = t - t.mean(-1, keepdim=True)
        return c / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-6)

    def rms(t, w=1.0):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6) * w

    phi = torch.cat([pos[..., c:c + 1].double() * 10000.0 ** (-torch.arange(0, d, 2).double() / d) for c, d in enumerate(AXES)], -1)
    cos, sin = phi.cos().unsqueeze(2), phi.sin().unsqueeze(2)

    def turn(t):
        t = t.unflatten(2, (HEADS, D))
        u, v = t[..., 0::2], t[..., 1::2]
        return torch.stack((u * cos - v * sin, u * sin + v * cos), -1).flatten(3)

    def attend(q, k, v, keys=None):
        s = torch.einsum("bqhd,bkhd->bhqk", q, k) / math.sqrt(D)
        if keys is not None:
            s = s.masked_fill(torch.arange(k.shape[1]) >= keys.view(-1, 1, 1, 1), -math.inf)
        return torch.einsum("bhqk,bkhd->bqhd", s.softmax(-1), v).flatten(2)

    heads = lambda t: t.unflatten(2, (HEADS, D))  # noqa: E731
    e = (p["table"] + p["time"]).unsqueeze(2)  # [B, 6, 1, C]
    y = layer(x) * (1 + e[:, 1]) + e[:, 0]
    a = attend(turn(rms(lin("q", y), p["qn"])), turn(rms(lin("k", y), p["kn"])), heads(lin("v", y)))
    x = x + lin("o", a) * e[:, 2]
    y = layer(x) * p["norm3_w"] + p["norm3_b"]
    a = attend(heads(rms(lin("cq", y), p["cqn"])), heads(rms(lin("ck", text), p["ckn"])), heads(lin("cv", text)), lengths)
    x = x + lin("co", a)
    y = lin("f2", torch.nn.functional.gelu(lin("f0", layer(x) * (1 + e[:, 4]) + e[:, 3]), approximate="tanh"))
    x = x + y * e[:, 5]
    return x, rms(x)


@pytest.mark.parametrize("dtype, tol_y, tol_g", [(torch.float32, 5e-5, 5e-5), (torch.bfloat16, 2e-2, 4e-2)])
def test_block_forward_and_gradients(pkg, dev, dtype, tol_y, tol_g):
    p = parameters(dtype, dev)
    lengths = torch.tensor([TXT, 5], dtype=torch.int32)
    pos = pkg.grid_positions([GRID, GRID], L)
    exact = {n: t.detach().double().cpu() for n, t in p.items()}
    for n in TRAINED:
        p[n].requires_grad_(True), exact[n].requires_grad_(True)
    outs = through_kernels(pkg, p, lengths.to(dev), pos.to(dev))
    want = exactly(exact, lengths, pos)
    g = torch.Generator().manual_seed(5)
    ups = [torch.randn(want[0].shape, generator=g).double() for _ in want]
    ups = [u.to(o.dtype).double() for u, o in zip(ups, outs)]
    grads = torch.autograd.grad(outs, [p[n] for n in TRAINED], [u.to(o.dtype).to(dev) for u, o in zip(ups, outs)])
    ref = torch.autograd.grad(want, [exact[n] for n in TRAINED], ups)
    rel = lambda a, b: float((a.detach().double().cpu() - b).norm() / b.norm())  # noqa: E731
    for i in range(2):
        assert rel(outs[i], want[i].detach()) <= tol_y, ("out", i, rel(outs[i], want[i].detach()))
    bad = {n: rel(a, b) for n, a, b in zip(TRAINED, grads, ref) if not rel(a, b) <= tol_g}
    assert not bad, bad


def test_block_captured_and_on_two_streams(pkg, dev):
    """The block's pass captured in a HIP graph and replayed with other inputs; two passes on two streams at once,
    their tensors made on a third: each equal to the eager pass on the default stream."""
    p = parameters(torch.bfloat16, dev)
    lengths = torch.tensor([TXT, 5], dtype=torch.int32, device=dev)
    pos = pkg.grid_positions([GRID, GRID], L, dev)
    for n in TRAINED:
        p[n].requires_grad_(True)
    leaves = [p[n] for n in TRAINED]

    def step():
        outs = through_kernels(pkg, p, lengths, pos)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, [torch.ones_like(o) for o in outs])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in range(3):
        with torch.no_grad():
            p["x"].copy_(torch.randn(p["x"].shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for _ in range(3):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append(step())
    torch.cuda.synchronize()
    for r in results:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(pkg, dev):
    """Samples more than 2^32 bytes apart, and a key cache whose tokens span more than 2^32 bytes."""
    far = (1 << 31) + 64
    big = torch.empty(far + 8 * 128, dtype=torch.bfloat16, device=dev)
    x = big.as_strided((2, 8, 128), (far, 128, 1))
    x.copy_(torch.randn(2, 8, 128))
    near = x.contiguous()
    y = torch.randn(2, 8, 128, device=dev).bfloat16()
    gate = torch.randn(2, 128, device=dev)
    for a, b in zip(pkg.gated_residual_norm(x, y, gate), pkg.gated_residual_norm(near, y, gate)):
        assert torch.equal(a, b)
    h, hn = x.unflatten(2, (2, 64)), near.unflatten(2, (2, 64))
    pos = torch.arange(16, device=dev, dtype=torch.int32).view(8, 2)
    assert torch.equal(pkg.rotary_axes(h, pos, (32, 32)), pkg.rotary_axes(hn, pos, (32, 32)))
    assert torch.equal(pkg.cross_attention(h, h, h), pkg.cross_attention(hn, hn, hn))
    del big, x, h
    wide = 1 << 21
    cache = torch.empty(1100 * wide, dtype=torch.bfloat16, device=dev)  # 4.6 GB
    k = cache.as_strided((1, 1100, 2, 64), (0, wide, 64, 1))
    v = cache.as_strided((1, 1100, 2, 64), (0, wide, 64, 1), 128)
    k.copy_(torch.randn(1, 1100, 2, 64)), v.copy_(torch.randn(1, 1100, 2, 64))
    kn, vn = k.contiguous(), v.contiguous()
    for rows in (3, 300):
        q = torch.randn(1, rows, 2, 64, device=dev).bfloat16()
        g = torch.randn(1, rows, 2, 64, device=dev).bfloat16()
        got, want = [], []
        for out, keys, values in ((got, k, v), (want, kn, vn)):
            leaves = [t.detach().requires_grad_(True) for t in (q, keys, values)]
            o = pkg.cross_attention(*leaves)
            out += [o.detach(), *torch.autograd.grad(o, leaves, [g])]
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_no_second_derivatives(pkg, dev):
    """A gradient that is differentiated again is refused, not wrong."""
    q = torch.randn(1, 4, 2, 32, device=dev, requires_grad=True)
    x = torch.randn(1, 4, 64, device=dev, requires_grad=True)
    pos = torch.arange(4, device=dev, dtype=torch.int32).view(4, 1)
    for leaf, out in ((q, pkg.cross_attention(q, q, q)), (q, pkg.rotary_axes(q, pos, (32,), weight=torch.ones(32, device=dev))),
                      (x, pkg.gated_residual_norm(x, x)[1])):
        d, = torch.autograd.grad(out.square().sum(), [leaf], create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            d.sum().backward()

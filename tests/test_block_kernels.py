"""The block operators' kernel calls (pkg.kernels), made without the operators in front of them: their own checks refuse what
the kernels would read out of range, and their results are the operators'."""
import pytest
import torch

BF, F = torch.bfloat16, torch.float32


def rotary_case(dev="cpu"):
    x, pos = torch.randn(2, 5, 4, 64).to(dev), torch.arange(10, dtype=torch.int32).view(1, 5, 2).to(dev)
    return dict(xs=[x, torch.randn(2, 5, 2, 64).to(dev)], positions=pos, axis_dims=(32, 32), theta=1e4, halves=False, eps=1e-6,
                norm=2, weights=[torch.ones(256).to(dev), torch.ones(128).to(dev)])


def test_rotary_refusals(pkg):
    K = pkg.kernels

    def bad(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            K.rotary_axes(**{**rotary_case(), **kw})

    c = rotary_case()
    x, k = c["xs"]
    bad("one or two", xs=[x] * 3)
    bad("one or two", xs=[x.half()])
    bad("one or two", xs=[x[0]])
    bad("must be torch.float32", xs=[x, k.to(BF)])
    bad("heads, head_dim", xs=[x, k[:1]])
    bad("one head_dim", xs=[x, k[..., :32].contiguous()])
    bad("16-byte", xs=[x.transpose(2, 3).contiguous().transpose(2, 3), k])
    for axes in ((32, 16), (32, 34), (31, 33), (), (-2, 66)):
        bad("axis_dims", axis_dims=axes)
    bad("norm is", norm=3)
    bad("for every tensor", weights=[torch.ones(256)])
    for w in ([torch.ones(256), torch.ones(64)], [torch.ones(64), torch.ones(64)], [torch.ones(256), None],
              [torch.ones(256), torch.ones(128).to(BF)], [torch.ones(256), torch.ones(128).half()], [torch.ones(256), torch.ones(256)[::2]]):
        bad("norm weights", weights=w)
    bad("norm weights", norm=1)
    for pos in (c["positions"][:, :4], c["positions"][..., :1], c["positions"][0], c["positions"].expand(3, 5, 2)):
        bad("positions must be", positions=pos)
    bad("positions must be", positions=c["positions"].to(torch.int16))
    bad("positions must be", positions=c["positions"].transpose(1, 2).contiguous().transpose(1, 2))
    bad("one ROCm device")

    def bad_backward(match, **kw):
        args = {**rotary_case(), "gs": [x, k], "want_dx": [True, True], "want_dw": [True, True], **kw}
        with pytest.raises(RuntimeError, match=match):
            K.rotary_axes_backward(**args)

    bad_backward("gradient for every", gs=[x])
    bad_backward("tensor's shape", gs=[x, x])
    bad_backward("must be torch.float32", gs=[x, k.to(BF)])
    bad_backward("norm weights", weights=[torch.ones(64), torch.ones(64)])
    bad_backward("axis_dims", axis_dims=(32, 16))
    bad_backward("one ROCm device")
    bad_backward("axis_dims", xs=None, norm=0, weights=(), want_dw=(), axis_dims=(32, 16))


def joint_case(dev="cpu", B=2):
    x = torch.randn(B, 5, 64).to(dev)
    v = lambda *s: torch.randn(*s).to(dev)  # noqa: E731
    return dict(x=x, y=x + 1, gate=v(B, 64), scale=v(64), shift=v(B, 1, 64), post_w=v(64), norm="layer", post="rms",
                unit_offset=True, alpha=1.0, eps=1e-6)


def test_joint_refusals(pkg):
    def bad(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.kernels.joint(**{**joint_case(), **kw})

    c = joint_case()
    bad("batch, tokens, width", x=c["x"][0])
    bad("x must be", x=c["x"].half())
    bad("y must be", y=c["y"][:, :4])
    bad("y must be", y=c["y"].transpose(1, 2).contiguous().transpose(1, 2))
    for v in (torch.ones(63), torch.ones(3, 64), torch.ones(2, 5, 64), torch.ones(64).half()):
        bad("gate must be", gate=v)
    bad("shared by the samples", post_w=torch.ones(2, 64))
    bad("share a dtype", shift=torch.ones(64).to(BF))
    bad("norm and post", norm="batch")
    bad("norm and post", post="none")
    bad("one ROCm device")

    def bad_backward(match, gx=c["x"], go=c["x"], **kw):
        args = {**joint_case(), **kw}
        with pytest.raises(RuntimeError, match=match):
            pkg.kernels.joint_backward(args.pop("x"), args.pop("y"), gx, go, **args, want=[True] * 6)

    bad_backward("gate must be", gate=torch.ones(63))
    bad_backward("one ROCm device")


def attention_case(dev="cpu"):
    r = lambda *s: torch.randn(*s).to(dev)  # noqa: E731
    return dict(q=r(2, 5, 4, 64), k=r(2, 7, 2, 64), v=r(2, 7, 2, 64), key_lengths=torch.tensor([7, 3], dtype=torch.int32).to(dev),
                key_mask=(torch.arange(7) != 2).view(1, 7).to(dev), scale=0.125)


def test_attention_refusals(pkg):
    def bad(match, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.kernels.cross_attention(**{**attention_case(), **kw})

    c = attention_case()
    bad("batch, tokens, heads", q=c["q"][0])
    bad("q must be", q=c["q"].half())
    bad("k must be", k=c["k"].to(BF))
    bad("v must be", v=c["v"][:, :6])
    bad("v must be", v=c["v"].transpose(2, 3).contiguous().transpose(2, 3))
    bad("key_lengths", key_lengths=c["key_lengths"].long())
    bad("key_lengths", key_lengths=c["key_lengths"][:1])
    bad("key_mask", key_mask=torch.ones(2, 6, dtype=torch.bool))
    bad("key_mask", key_mask=torch.ones(7, dtype=torch.bool))
    bad("key_mask", key_mask=torch.ones(7, 2, dtype=torch.bool).t())
    bad("one ROCm device")


def same(got, want):
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_results_are_the_operators(pkg, dev):
    K = pkg.kernels
    c = rotary_case(dev)
    leaves = [t.requires_grad_(True) for t in (*c["xs"], *c["weights"])]
    outs = pkg.rotary_axes_qk(*leaves[:2], c["positions"], c["axis_dims"], q_weight=leaves[2], k_weight=leaves[3])
    gs = [torch.randn_like(o) for o in outs]
    want = torch.autograd.grad(outs, leaves, gs)
    with torch.no_grad():
        same(K.rotary_axes(**c), outs)
        dxs, dws = K.rotary_axes_backward(**c, gs=gs, want_dx=[True, True], want_dw=[True, True])
    same([*dxs, *dws], want)

    c = joint_case(dev)
    names = ("x", "y", "gate", "scale", "shift", "post_w")
    leaves = [c[n].requires_grad_(True) for n in names]
    outs = pkg.gated_residual_norm(*leaves[:5], post_norm="rms", post_weight=leaves[5])
    gs = [torch.randn_like(o) for o in outs]
    want = torch.autograd.grad(outs, leaves, gs)
    with torch.no_grad():
        same(K.joint(**c), outs)
        kw = dict(norm="layer", post="rms", unit_offset=True, alpha=1.0, eps=1e-6, want=[True] * 6)
        same(K.joint_backward(*leaves[:2], *gs, *leaves[2:], **kw), want)
        for t in (gs[0][:, :4], gs[0].to(BF), gs[0].cpu()):
            with pytest.raises(RuntimeError, match="kernel contract"):
                K.joint_backward(*leaves[:2], t, gs[1], *leaves[2:], **kw)

    c = attention_case(dev)
    leaves = [c[n].requires_grad_(True) for n in ("q", "k", "v")]
    out = pkg.cross_attention(*leaves, key_lengths=c["key_lengths"], key_mask=c["key_mask"])
    g = torch.randn_like(out)
    want = torch.autograd.grad(out, leaves, [g])
    with torch.no_grad():
        got, lse = K.cross_attention(**c)
        same([got], [out])
        same(K.cross_attention_backward(out=out, lse=lse, g=g, **c), want)
        for kw in (dict(g=g[:, :4]), dict(g=g.to(BF)), dict(lse=lse[:1]), dict(lse=lse.double()), dict(out=out.transpose(0, 1).contiguous().transpose(0, 1)),
                   dict(g=g.cpu()), dict(lse=lse.cpu())):
            with pytest.raises(RuntimeError, match="kernel contract"):
                K.cross_attention_backward(**{**dict(out=out, lse=lse, g=g, **c), **kw})

"""What the operators between a block's linears refuse, and their C entries' checks before any launch (no
GPU needed)."""
import ctypes

import pytest
import torch

BF, F = torch.bfloat16, torch.float32


def test_grid_positions(pkg):
    pos = pkg.grid_positions(torch.tensor([[2, 2, 3], [1, 1, 1]]), 13)
    assert pos.dtype == torch.int32 and pos.shape == (2, 13, 3)
    assert pos[0, :12].tolist() == [[f, h, w] for f in range(2) for h in range(2) for w in range(3)]
    assert pos[0, 12].tolist() == [0, 0, 0] and pos[1].abs().sum() == 0
    assert pkg.grid_positions([[2, 2]], 4, start=(3, 1))[0].tolist() == [[3, 1], [3, 2], [4, 1], [4, 2]]
    assert pkg.grid_positions([[0, 2]], 3).abs().sum() == 0
    for bad in ([[3, 2]], [[-1, 2]], [], [[1, 2], [1]]):
        with pytest.raises(RuntimeError, match="rotary axes"):
            pkg.grid_positions(bad, 5)
    with pytest.raises(RuntimeError, match="start"):
        pkg.grid_positions([[1, 2]], 5, start=(1, 2, 3))


def test_rotary_refusals(pkg):
    x, pos = torch.zeros(2, 5, 4, 64), torch.zeros(5, 2, dtype=torch.int32)

    def bad(match, x=x, pos=pos, axes=(32, 32), **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.rotary_axes(x, pos, axes, **kw)

    bad("batch, tokens", x=x[0])
    bad("bfloat16 or float32", x=x.half())
    bad("multiple of 16", x=torch.zeros(2, 5, 4, 40), axes=(20, 20))
    bad("multiple of 16", x=torch.zeros(2, 5, 4, 272), axes=(136, 136))
    bad("8192", x=torch.zeros(1, 5, 129, 64))
    bad("8192", x=torch.zeros(1, 5, 0, 64))
    for axes in ((32, 30), (31, 33), (), (-2, 66)):
        bad("axis_dims", axes=axes)
    bad("pairing", pairing="split")
    bad("theta", theta=0.0)
    bad("eps", eps=0.0)
    bad("positions", pos=pos.to(torch.int16))
    bad("positions", pos=torch.zeros(5, 3, dtype=torch.int32))
    bad("positions", pos=torch.zeros(3, 5, 2, dtype=torch.int32))
    bad("no gradient", pos=torch.zeros(5, 2, requires_grad=True))
    bad("weight", weight=torch.ones(63))
    bad("weight", weight=torch.ones(64).half())
    bad("ROCm device", weight=torch.ones(64))
    k = torch.zeros(2, 5, 2, 64)

    def bad_qk(match, q=x, k=k, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.rotary_axes_qk(q, k, pos, (32, 32), **kw)

    bad_qk("one dtype", k=k.to(BF))
    bad_qk("share batch", k=k[:1])
    bad_qk("come together", q_weight=torch.ones(64))
    bad_qk("normed alike", q_weight=torch.ones(256), k_weight=torch.ones(64))
    bad_qk("share a dtype", q_weight=torch.ones(64), k_weight=torch.ones(64).to(BF))
    bad_qk("ROCm device", k=k[:, :, :1], q_weight=torch.ones(256), k_weight=torch.ones(64))  # one head: its row


def test_joint_refusals(pkg):
    x = torch.zeros(2, 5, 64)

    def bad(match, x=x, y=x, *vectors, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.gated_residual_norm(x, y, *vectors, **kw)

    bad("batch, tokens", x=x[0])
    bad("bfloat16 or float32", y=x.half())
    bad("share shape", y=x[:1])
    bad("bfloat16 stream", x=x.to(BF))
    bad("multiple of 8", x=torch.zeros(1, 2, 60), y=torch.zeros(1, 2, 60))
    bad("multiple of 8", x=torch.zeros(1, 1, 8200), y=torch.zeros(1, 1, 8200))
    bad("norm", norm="batch")
    bad("norm", post_norm="none")
    bad("needs a post_norm", post_weight=torch.ones(64))
    bad("needs a scale", shift=torch.ones(64))
    bad("eps", eps=float("nan"))
    bad("residual_scale", residual_scale=float("inf"))
    for v in (torch.ones(63), torch.ones(3, 64), torch.ones(2, 5, 64), torch.ones(64).half()):
        bad("gate", gate=v)
    bad("post_weight", post_norm="rms", post_weight=torch.ones(2, 64))
    bad("share a dtype", scale=torch.ones(64), shift=torch.ones(64).to(BF))
    bad("ROCm device", gate=torch.ones(2, 1, 64))


def test_rotary_entries_validate_before_launch(pkg):
    L, lib = pkg._lib, pkg._lib.load()
    turns, axis = (ctypes.c_double * 32)(), (ctypes.c_int32 * 32)()
    assert lib.mlora_rotary_turns(L.i32_array([24, 40]), 2, 10000.0, turns, axis) == L.OK
    assert list(axis) == [0] * 12 + [1] * 20 and abs(turns[1] * 2 * 3.141592653589793 - 10000 ** (-2 / 24)) < 1e-15
    assert lib.mlora_rotary_turns(L.i32_array([24, 41]), 2, 10000.0, turns, axis) == L.ERR_INVALID
    assert lib.mlora_rotary_turns(L.i32_array([24, 40]), 2, -1.0, turns, axis) == L.ERR_INVALID
    assert lib.mlora_rotary_turns(L.i32_array([258]), 1, 1e4, turns, axis) == L.ERR_LIMIT

    def fwd(x=0x1000, y=0x2000, w=0x3000, strides=(20480, 256, 64), heads=4, n=1, dt=L.BF16, wdt=L.F32, norm=1, eps=1e-6,
            pos=0x4000, kind=0, n_axes=2, B=2, T=5, D=64, t=turns):
        return lib.mlora_rotary_axes(L.ptr_array([x]), L.ptr_array([y]), L.ptr_array([w]), L.i64_array(strides),
                                     L.i32_array([heads]), n, dt, wdt, norm, eps, pos, kind, 0, 2, t, axis, n_axes, 0,
                                     B, T, D, None)

    assert fwd(B=0) == L.OK
    for kw, code in ((dict(x=0), L.ERR_INVALID), (dict(x=0x1008), L.ERR_UNSUPPORTED), (dict(y=0), L.ERR_INVALID),
                     (dict(y=0x2004), L.ERR_UNSUPPORTED), (dict(w=0), L.ERR_INVALID), (dict(strides=(20480, 252, 64)), L.ERR_UNSUPPORTED),
                     (dict(strides=(20480, 256, -64)), L.ERR_UNSUPPORTED), (dict(heads=0), L.ERR_INVALID), (dict(heads=129), L.ERR_LIMIT),
                     (dict(n=3), L.ERR_INVALID), (dict(dt=L.FP8_E4M3), L.ERR_UNSUPPORTED), (dict(norm=3), L.ERR_INVALID),
                     (dict(eps=0.0), L.ERR_INVALID), (dict(pos=0), L.ERR_INVALID), (dict(kind=3), L.ERR_INVALID),
                     (dict(n_axes=1), L.ERR_INVALID), (dict(D=60), L.ERR_UNSUPPORTED), (dict(D=272), L.ERR_UNSUPPORTED),
                     (dict(B=1 << 20, T=1 << 12), L.ERR_LIMIT), (dict(T=-1), L.ERR_INVALID), (dict(t=None), L.ERR_INVALID)):
        assert fwd(**kw) == code, kw
    heads = L.i32_array([4, 2])
    ws = lambda norm, B=2, T=5: lib.mlora_rotary_axes_backward_workspace_bytes(heads, 2, norm, B, T, 64)  # noqa: E731
    assert ws(0) == 0 and ws(1) == 3 * 2 * 64 * 4 and ws(2) == 3 * 6 * 64 * 4 and ws(2, T=0) == 0  # 10 rows, 4 to a workgroup
    assert ws(1, B=-1) == L.ERR_INVALID and ws(1, 1 << 20, 1 << 12) == L.ERR_LIMIT

    def bwd(g=0x5000, dx=0x6000, dw=0x7000, work=0x8000, nbytes=3 * 64 * 4, norm=1, x=0x1000):
        return lib.mlora_rotary_axes_backward(L.ptr_array([x]), L.ptr_array([g]), L.ptr_array([dx]), L.ptr_array([0x3000]),
                                              L.ptr_array([dw]), L.i64_array([20480, 256, 64]), L.i64_array([20480, 256, 64]),
                                              L.i32_array([4]), 1, L.BF16, L.F32, norm, 1e-6, 0x4000, 0, 0, 2, turns, axis, 2,
                                              0, work, nbytes, 2, 5, 64, None)

    assert bwd(nbytes=3 * 64 * 4 - 1) == L.ERR_WORKSPACE and bwd(work=0) == L.ERR_WORKSPACE
    assert bwd(work=0x8004) == L.ERR_UNSUPPORTED and bwd(g=0) == L.ERR_INVALID and bwd(g=0x5002) == L.ERR_UNSUPPORTED
    assert bwd(norm=0) == L.ERR_INVALID and bwd(x=0) == L.ERR_INVALID and bwd(dx=0x6004) == L.ERR_UNSUPPORTED
    assert bwd(dw=0x7002) == L.ERR_UNSUPPORTED


def test_joint_entries_validate_before_launch(pkg):
    L, lib = pkg._lib, pkg._lib.load()

    def args(x=0x1000, xdt=L.F32, xst=64, y=0x2000, ydt=L.BF16, gate=0x3000, gsb=64, scale=0x4000, shift=0x5000,
             adt=L.F32, post_w=None, norm=0, post=-1, alpha=1.0, eps=1e-6):
        return ((x, xdt, 320, xst, y, ydt, 320, 64),
                (gate, L.F32, gsb, scale, shift, adt, 64, 64, 1, post_w, L.F32, norm, post, alpha, eps))

    def fwd(x1=0x6000, out=0x7000, B=2, T=5, W=64, **kw):
        head, tail = args(**kw)
        return lib.mlora_joint(*head, *tail, x1, out, B, T, W, None)

    assert fwd(T=0) == L.OK and fwd(W=0) == L.OK
    for kw, code in ((dict(x=0), L.ERR_INVALID), (dict(x=0x1004), L.ERR_UNSUPPORTED), (dict(xst=60), L.ERR_UNSUPPORTED),
                     (dict(xdt=L.BF16, ydt=L.F32), L.ERR_UNSUPPORTED), (dict(gsb=4), L.ERR_UNSUPPORTED),
                     (dict(scale=0), L.ERR_INVALID), (dict(post_w=0x9000), L.ERR_INVALID), (dict(norm=2), L.ERR_INVALID),
                     (dict(post=2), L.ERR_INVALID), (dict(alpha=float("nan")), L.ERR_INVALID), (dict(eps=0.0), L.ERR_INVALID),
                     (dict(adt=7), L.ERR_UNSUPPORTED), (dict(W=60), L.ERR_UNSUPPORTED), (dict(W=8200), L.ERR_UNSUPPORTED),
                     (dict(B=1 << 20, T=1 << 12), L.ERR_LIMIT), (dict(B=-1), L.ERR_INVALID), (dict(x1=0), L.ERR_INVALID),
                     (dict(out=0x7008), L.ERR_UNSUPPORTED)):
        assert fwd(**kw) == code, kw
    ws = lib.mlora_joint_backward_workspace_bytes(2, 5, 64)
    assert ws == 2 * 2 * 4 * 64 * 4  # two workgroups of four rows per sample, four vectors
    assert lib.mlora_joint_backward_workspace_bytes(2, 0, 64) == 0
    assert lib.mlora_joint_backward_workspace_bytes(2, 5, 8200) == L.ERR_UNSUPPORTED

    def bwd(dgate=0xa000, dscale=0xb000, dpost=None, work=0xc000, nbytes=ws, gx=0x8000, dx=0x9000, **kw):
        head, tail = args(**kw)
        return lib.mlora_joint_backward(*head, gx, 320, 64, 0xd000, 320, 64, *tail, dx, 0xe000, dgate, dscale, None, dpost,
                                        0, 0, 0, work, nbytes, 2, 5, 64, None)

    assert bwd(nbytes=ws - 1) == L.ERR_WORKSPACE and bwd(work=0) == L.ERR_WORKSPACE and bwd(work=0xc004) == L.ERR_UNSUPPORTED
    assert bwd(gate=0) == L.ERR_INVALID and bwd(dpost=0xf000) == L.ERR_INVALID
    assert bwd(gx=0x8004) == L.ERR_UNSUPPORTED and bwd(dx=0x9008) == L.ERR_UNSUPPORTED


def test_attention_refusals(pkg):
    q, k = torch.zeros(2, 5, 4, 64), torch.zeros(2, 7, 2, 64)

    def bad(match, q=q, k=k, v=None, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.cross_attention(q, k, k if v is None else v, **kw)

    bad("batch, tokens", q=q[0])
    bad("bfloat16 or float32", q=q.half())
    bad("one dtype", k=k.to(BF))
    bad("k and v must be", v=k[:, :6])
    bad("k and v must be", k=k[:1])
    bad("k and v must be", k=torch.zeros(2, 7, 2, 32))
    bad("share", k=torch.zeros(2, 7, 3, 64))
    bad("share", k=torch.zeros(2, 7, 0, 64))
    bad("multiple of 8", q=torch.zeros(2, 5, 4, 60), k=torch.zeros(2, 7, 2, 60))
    bad("multiple of 8", q=torch.zeros(2, 5, 4, 136), k=torch.zeros(2, 7, 2, 136))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        bad("scale", scale=scale)
    bad("key_lengths", key_lengths=torch.zeros(2))
    bad("key_lengths", key_lengths=torch.zeros(3, dtype=torch.int32))
    bad("key_mask", key_mask=torch.zeros(2, 7, dtype=torch.uint8))
    bad("key_mask", key_mask=torch.zeros(2, 6, dtype=torch.bool))
    bad("ROCm device", key_lengths=torch.zeros(2, dtype=torch.int64), key_mask=torch.zeros(7, dtype=torch.bool))


def test_attention_entries_validate_before_launch(pkg):
    L, lib = pkg._lib, pkg._lib.load()
    st = (1280, 256, 64)

    def fwd(q=0x1000, k=0x2000, v=0x3000, qs=st, ks=st, dt=L.BF16, mask=None, mask_sb=0, scale=0.125, out=0x4000, lse=0x5000,
            work=0x6000, nbytes=1 << 30, B=2, Lq=5, Lk=7, H=4, Hk=4, D=64):
        return lib.mlora_cross_attention(q, L.i64_array(qs), k, L.i64_array(ks), v, L.i64_array(st), dt, None, mask, mask_sb,
                                         scale, out, lse, work, nbytes, B, Lq, Lk, H, Hk, D, None)

    assert fwd(B=0) == L.OK and fwd(Lq=0, q=0, out=0, lse=0) == L.OK
    for kw, code in ((dict(q=0), L.ERR_INVALID), (dict(q=0x1008), L.ERR_UNSUPPORTED), (dict(k=0), L.ERR_INVALID),
                     (dict(qs=(1280, 252, 64)), L.ERR_UNSUPPORTED), (dict(qs=(1280, -256, 64)), L.ERR_UNSUPPORTED),
                     (dict(ks=(1280, 1 << 22, 64)), L.ERR_LIMIT), (dict(dt=L.FP8_E4M3), L.ERR_UNSUPPORTED),
                     (dict(mask=0x7000, mask_sb=-1), L.ERR_INVALID), (dict(scale=0.0), L.ERR_INVALID),
                     (dict(scale=float("inf")), L.ERR_INVALID), (dict(out=0), L.ERR_INVALID), (dict(out=0x4004), L.ERR_UNSUPPORTED),
                     (dict(lse=0), L.ERR_INVALID), (dict(lse=0x5002), L.ERR_UNSUPPORTED), (dict(Hk=3), L.ERR_INVALID),
                     (dict(H=0), L.ERR_INVALID), (dict(D=60), L.ERR_UNSUPPORTED), (dict(D=136), L.ERR_UNSUPPORTED),
                     (dict(Lk=1 << 31), L.ERR_LIMIT), (dict(Lq=1 << 30, H=8, Hk=1), L.ERR_LIMIT), (dict(Lq=-1), L.ERR_INVALID),
                     (dict(B=1 << 20, Lq=1 << 24), L.ERR_LIMIT)):
        assert fwd(**kw) == code, kw
    # few rows against many keys: partial sums need a workspace
    size = lambda *a: lib.mlora_cross_attention_workspace_bytes(L.BF16, *a)  # noqa: E731
    need = size(1, 1, 4096, 4, 4, 64)
    assert need > 0 and need % ((64 + 2) * 4 * 4) == 0 and size(1, 4096, 64, 4, 4, 64) == 0 and size(1, 1, 0, 4, 4, 64) == 0
    assert size(1, 1, 4096, 4, 3, 64) == L.ERR_INVALID
    assert fwd(B=1, Lq=1, Lk=4096, nbytes=need - 1) == L.ERR_WORKSPACE and fwd(B=1, Lq=1, Lk=4096, work=0) == L.ERR_WORKSPACE
    assert fwd(B=1, Lq=1, Lk=4096, work=0x6004) == L.ERR_UNSUPPORTED
    back = lib.mlora_cross_attention_backward_workspace_bytes(L.BF16, 2, 5, 7, 4, 4, 64)
    assert back >= 2 * 4 * 5 * 4

    def bwd(g=0x7000, gs=st, dq=0x8000, dk=0x9000, out=0x4000, work=0x6000, nbytes=back, lse=0x5000):
        return lib.mlora_cross_attention_backward(0x1000, L.i64_array(st), 0x2000, L.i64_array(st), 0x3000, L.i64_array(st),
                                                  L.BF16, None, None, 0, 0.125, out, lse, g, L.i64_array(gs), dq, dk, 0xa000,
                                                  work, nbytes, 2, 5, 7, 4, 4, 64, None)

    assert bwd(g=0) == L.ERR_INVALID and bwd(gs=(1280, 252, 64)) == L.ERR_UNSUPPORTED and bwd(dq=0) == L.ERR_INVALID
    assert bwd(dk=0) == L.ERR_INVALID and bwd(dk=0x9004) == L.ERR_UNSUPPORTED and bwd(out=0) == L.ERR_INVALID
    assert bwd(lse=0) == L.ERR_INVALID and bwd(nbytes=back - 1) == L.ERR_WORKSPACE and bwd(work=0) == L.ERR_WORKSPACE
    assert bwd(work=0x6008) == L.ERR_UNSUPPORTED

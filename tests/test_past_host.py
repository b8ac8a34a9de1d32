"""What window_attention and prefix_attention refuse, and their C entries' checks before any launch (no GPU needed)."""
import ctypes

import pytest
import torch

import past_plans

BF, F = torch.bfloat16, torch.float32


def heads(B=2, L=5, H=4, D=64, dtype=F):
    return torch.zeros(B, L, H, D, dtype=dtype)


def test_window_refusals(pkg):
    q, k = heads(), heads(L=7, H=2)

    def bad(match, q=q, k=k, v=None, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.window_attention(q, k, k if v is None else v, **kw)

    bad("batch, tokens", q=q[0])
    bad("batch, tokens", k=k[0])
    bad("bfloat16 or float32", q=q.half())
    bad("one dtype", k=k.to(BF))
    bad("k and v must be", v=k[:, :6])
    bad("k and v must be", k=k[:1])
    bad("k and v must be", k=heads(L=7, H=2, D=32))
    bad("share", k=heads(L=7, H=3))
    bad("share", k=heads(L=7, H=0))
    bad("share", q=heads(H=0), k=heads(L=7, H=0))
    bad("multiple of 8", q=heads(D=60), k=heads(L=7, H=2, D=60))
    bad("multiple of 8", q=heads(D=136), k=heads(L=7, H=2, D=136))
    bad("chunk", chunk=0)
    bad("window", window=0)
    bad("window", window=3, chunk=4)
    bad("sinks", sinks=-1)
    for name in ("window", "sinks", "chunk", "query_start"):
        bad(name, **{name: 2.5})
        bad(name, **{name: "many"})
        bad(name, **{name: float("nan")})
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        bad("scale", scale=scale)
    bad("no gradient", scale=torch.tensor(0.5, requires_grad=True))
    bad("give query_start", q=heads(L=9))
    for name in ("key_lengths", "query_start"):
        bad(name, **{name: torch.zeros(2)})
        bad(name, **{name: torch.zeros(3, dtype=torch.int32)})
        bad(name, **{name: torch.zeros(2, 1, dtype=torch.int32)})
    bad("must be a tensor", key_lengths=[5, 5])
    bad("must be a tensor", v=[1.0])
    bad("at most", q=heads(B=1, L=1), k=torch.zeros(1, 1, 2, 64).expand(1, (1 << 28) + 1, 2, 64))
    bad("ROCm device", window=2, sinks=3, chunk=2, key_lengths=torch.zeros(2, dtype=torch.int64), query_start=-1)


def test_prefix_refusals(pkg):
    q, k, p = heads(B=4), heads(B=4, L=7, H=2), heads(L=9, H=2)

    def bad(match, pk=p, pv=None, **kw):
        with pytest.raises(RuntimeError, match=match):
            pkg.prefix_attention(q, k, k, pk, pk if pv is None else pv, **kw)

    bad("share 3 prefixes", pk=heads(B=3, L=9, H=2))
    bad("share 0 prefixes", pk=heads(B=0, L=9, H=2))
    bad("prefix_k and prefix_v must be", pv=p[:, :8])
    bad("prefix_k and prefix_v must be", pv=p[0])
    bad("prefix_k and prefix_v must be", pk=heads(L=9, H=4))
    bad("prefix_k and prefix_v must be", pk=heads(L=9, H=2, D=32))
    bad("prefix_k and prefix_v must be", pk=p[0, 0], pv=p[0, 0])
    bad("dtype and device", pk=p.to(BF))
    bad("dtype and device", pv=p.to(BF))
    bad("prefix_lengths", prefix_lengths=torch.zeros(4, dtype=torch.int32))
    bad("prefix_lengths", prefix_lengths=torch.zeros(2))
    bad("ROCm device", prefix_lengths=torch.zeros(2, dtype=torch.int64), window=3)
    bad("ROCm device", pk=p[0])


def test_forward_mode_is_refused(pkg, monkeypatch):
    """A tangent is never dropped without a word; without one the same call reaches the kernel."""
    from torch.autograd import forward_ad

    reached = []
    monkeypatch.setattr(pkg.past_attention, "_plan", lambda *a: (None, a[1:]))
    monkeypatch.setattr(pkg.past_attention, "_lay_out", lambda call, tensors: (None, tensors, []))
    monkeypatch.setattr(pkg.kernels, "past_attention", lambda *a: (reached.append(a), (None, None))[1])
    q = heads()
    for at in range(3):
        with forward_ad.dual_level(), torch.no_grad():
            tensors = [forward_ad.make_dual(q, torch.ones_like(q)) if i == at else q for i in range(3)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                pkg.window_attention(*tensors)
    pkg.window_attention(q, q, q)
    assert len(reached) == 1


def shape(L, **kw):
    d = dict(dtype=L.BF16, from_end=0, B=2, Lq=5, Lk=7, H=4, Hk=4, D=64, groups=0, Lp=0, window=0, sinks=0, chunk=1, first=2,
             q=(1280, 256, 64), k=(1792, 256, 64), v=(1792, 256, 64), pk=(0, 0, 0), pv=(0, 0, 0), scale=0.125)
    d.update(kw)
    strides = [(ctypes.c_int64 * 3)(*d.pop(n)) for n in ("q", "k", "v", "pk", "pv")]
    scale = d.pop("scale")
    return ctypes.byref(L.PastShape(*d.values(), *strides, scale))


BAD_SHAPES = [
    (dict(dtype=2), "ERR_UNSUPPORTED"), (dict(B=-1), "ERR_INVALID"), (dict(Lq=-1), "ERR_INVALID"), (dict(Lk=-1), "ERR_INVALID"),
    (dict(H=0), "ERR_INVALID"), (dict(Hk=0), "ERR_INVALID"), (dict(Hk=3), "ERR_INVALID"), (dict(D=60), "ERR_UNSUPPORTED"),
    (dict(D=0), "ERR_UNSUPPORTED"), (dict(D=136), "ERR_UNSUPPORTED"), (dict(window=-1), "ERR_INVALID"), (dict(sinks=-1), "ERR_INVALID"),
    (dict(chunk=0), "ERR_INVALID"), (dict(window=3, chunk=4), "ERR_INVALID"), (dict(groups=-1), "ERR_INVALID"),
    (dict(groups=3), "ERR_INVALID"), (dict(Lp=4), "ERR_INVALID"), (dict(groups=1, Lp=-1), "ERR_INVALID"), (dict(scale=0.0), "ERR_INVALID"),
    (dict(scale=float("inf")), "ERR_INVALID"), (dict(scale=3e38), "ERR_INVALID"), (dict(Lk=(1 << 28) + 1), "ERR_LIMIT"),
    (dict(Lq=(1 << 28) + 1), "ERR_LIMIT"), (dict(groups=1, Lp=(1 << 28) + 1), "ERR_LIMIT"), (dict(H=1 << 17), "ERR_LIMIT"),
    (dict(Lq=1 << 28, H=16, Hk=1), "ERR_LIMIT"), (dict(B=1 << 24, Lk=1 << 20), "ERR_LIMIT"), (dict(B=1 << 40), "ERR_LIMIT"),
]


@pytest.mark.parametrize("case", BAD_SHAPES, ids=str)
def test_entries_refuse_sizes(pkg, case):
    L, lib = pkg._lib, pkg._lib.load()
    kw, code = case
    s, code = shape(L, **kw), getattr(L, code)
    assert lib.mlora_past_attention_workspace_bytes(s) == code and lib.mlora_past_attention_backward_workspace_bytes(s) == code
    ptr = [0x1000] * 5
    assert lib.mlora_past_attention(s, *ptr, None, None, None, 0x2000, 0x3000, 0x4000, 0x5000, 1 << 40, None) == code
    assert lib.mlora_past_attention_backward(s, *ptr, None, None, None, 0x2000, 0x3000, 0x4000, 0x6000,
                                             (ctypes.c_int64 * 3)(1280, 256, 64), *[0x7000] * 5, 0x5000, 1 << 40, None) == code


def test_entries_validate_before_launch(pkg):
    L, lib = pkg._lib, pkg._lib.load()

    def fwd(q=0x1000, k=0x2000, v=0x3000, pk=None, pv=None, out=0x4000, rest=0x5000, stats=0x6000, work=0x7000, nbytes=1 << 40, **kw):
        return lib.mlora_past_attention(shape(L, **kw), q, k, v, pk, pv, None, None, None, out, rest, stats, work, nbytes, None)

    assert lib.mlora_past_attention_workspace_bytes(None) == L.ERR_INVALID
    assert fwd(B=0) == L.OK and fwd(Lq=0, q=None, out=None, rest=None, stats=None) == L.OK
    group = dict(groups=1, Lp=4, pk=0x8000, pv=0x9000)
    for kw, code in ((dict(q=None), L.ERR_INVALID), (dict(q=0x1008), L.ERR_UNSUPPORTED), (dict(k=None), L.ERR_INVALID),
                     (dict(v=0x3004), L.ERR_UNSUPPORTED), (dict(out=None), L.ERR_INVALID), (dict(out=0x4008), L.ERR_UNSUPPORTED),
                     (dict(rest=None), L.ERR_INVALID), (dict(rest=0x5002), L.ERR_UNSUPPORTED), (dict(stats=0x6002), L.ERR_UNSUPPORTED),
                     (dict(group, pk=None), L.ERR_INVALID), (dict(group, pv=0x9008), L.ERR_UNSUPPORTED)):
        kw = dict(kw)
        pk, pv = kw.pop("pk", None), kw.pop("pv", None)
        strides = {}
        if "groups" in kw:
            strides = dict(groups=kw.pop("groups"), Lp=kw.pop("Lp"))
            s = shape(L, **strides, pk=(1024, 256, 64), pv=(1024, 256, 64))
            assert lib.mlora_past_attention(s, 0x1000, 0x2000, 0x3000, pk, pv, None, None, None, 0x4000, 0x5000, 0x6000, 0x7000, 1 << 40,
                                            None) == code, kw
        else:
            assert fwd(**kw) == code, kw
    for name, index in (("q", 0), ("k", 0), ("v", 0)):
        for strides, code in (((1280, 252, 64), L.ERR_UNSUPPORTED), ((1280, -256, 64), L.ERR_UNSUPPORTED), ((1280, 256, 60), L.ERR_UNSUPPORTED),
                              ((1284, 256, 64), L.ERR_UNSUPPORTED), ((1280, 1 << 22, 64), L.ERR_LIMIT)):
            s = shape(L, **{name: strides})
            assert lib.mlora_past_attention(s, 0x1000, 0x2000, 0x3000, None, None, None, None, None, 0x4000, 0x5000, 0x6000, 0x7000, 1 << 40,
                                            None) == code, (name, strides)


def test_workspaces(pkg):
    """Shares of the keys need a workspace, the backward its deltas; one byte less is refused."""
    L, lib = pkg._lib, pkg._lib.load()
    token = dict(B=1, Lq=1, Lk=4096, first=4095)
    need = lib.mlora_past_attention_workspace_bytes(shape(L, **token))
    assert need > 0 and need % ((64 + 2) * 4 * 4) == 0
    assert lib.mlora_past_attention_workspace_bytes(shape(L, B=1, Lq=4096, Lk=64)) == 0
    for empty in (dict(B=0), dict(Lq=0), dict(Lk=0), dict(B=0, Lq=0, Lk=0), dict(Lq=0, groups=1, Lp=1 << 20, Lk=1 << 20)):
        assert lib.mlora_past_attention_workspace_bytes(shape(L, **empty)) >= 0
        assert lib.mlora_past_attention_backward_workspace_bytes(shape(L, **empty)) >= 0

    def fwd(work=0x7000, nbytes=need):
        return lib.mlora_past_attention(shape(L, **token), 0x1000, 0x2000, 0x3000, None, None, None, None, None, 0x4000, None, None, work,
                                        nbytes, None)

    assert fwd(nbytes=need - 1) == L.ERR_WORKSPACE and fwd(work=None) == L.ERR_WORKSPACE and fwd(work=0x7008) == L.ERR_UNSUPPORTED
    # windows, sinks and chunks of any size mean what they mean at the number of keys
    for kw in (dict(window=1 << 62), dict(sinks=1 << 62), dict(window=1 << 62, chunk=1 << 62)):
        assert lib.mlora_past_attention_workspace_bytes(shape(L, **token, **kw)) == need
    back = lib.mlora_past_attention_backward_workspace_bytes(shape(L))
    assert back >= 2 * 4 * 5 * 4

    def bwd(g=0x8000, gs=(1280, 256, 64), out=0x4000, rest=0x5000, stats=0x6000, dq=0x9000, dk=0xa000, dv=0xb000, work=0x7000, nbytes=back):
        return lib.mlora_past_attention_backward(shape(L), 0x1000, 0x2000, 0x3000, None, None, None, None, None, out, rest, stats, g,
                                                 gs if gs is None else (ctypes.c_int64 * 3)(*gs), dq, dk, dv, None, None, work, nbytes, None)

    for kw, code in ((dict(g=None), L.ERR_INVALID), (dict(gs=None), L.ERR_INVALID), (dict(gs=(1280, 252, 64)), L.ERR_UNSUPPORTED),
                     (dict(out=None), L.ERR_INVALID), (dict(rest=None), L.ERR_INVALID), (dict(stats=None), L.ERR_INVALID),
                     (dict(dq=None), L.ERR_INVALID), (dict(dk=None), L.ERR_INVALID), (dict(dv=0xb008), L.ERR_UNSUPPORTED),
                     (dict(work=None), L.ERR_WORKSPACE), (dict(nbytes=back - 1), L.ERR_WORKSPACE), (dict(work=0x7004), L.ERR_UNSUPPORTED)):
        assert bwd(**kw) == code, kw


@pytest.fixture
def on_device(pkg, monkeypatch):
    """Host tensors pass for device tensors."""
    meta = pkg.past_attention._meta

    def moved(*a):
        m = meta(*a)
        return m and (*m[:2], torch.device("cuda", 0), *m[3:])

    monkeypatch.setattr(pkg.past_attention, "_meta", moved)


@pytest.fixture
def told(pkg, on_device, monkeypatch):
    """The operators up to their launches, on host tensors: what kernels.past_attention_backward is called with, call by call."""
    calls = []

    def forward(plan, tensors, pointers, *rest):
        return torch.zeros(tensors[0].shape, dtype=tensors[0].dtype), torch.zeros(plan.saved)

    def backward(plan, out, saved, g, tensors, *vectors):
        calls.append((plan, out, saved, g, tensors, vectors))
        return [torch.zeros(t.shape, dtype=t.dtype) for t in tensors]

    monkeypatch.setattr(pkg.kernels, "past_attention", forward)
    monkeypatch.setattr(pkg.kernels, "past_attention_backward", backward)
    return calls


def strided_last(t):
    return torch.stack((t, t), dim=-1).flatten(-2)[..., ::2]


def misaligned(t):
    return torch.cat((t.new_zeros(1), t.reshape(-1)))[1:].view(t.shape)


HOOKS = {
    "contiguous": lambda t: t.clone(memory_format=torch.contiguous_format),
    "clone": torch.clone,
    "reversed": lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim()))),
    "strided last": strided_last,
    "misaligned": misaligned,
    "as it was": lambda t: t,
}


def operands(dtype, prefix):
    """q, k and v of packed projections, head-major and expanded storage."""
    r = lambda *s: torch.randn(*s, generator=torch.Generator().manual_seed(len(s) + s[1])).to(dtype)  # noqa: E731
    t = [r(2, 50, 3, 4, 64)[:, :, 0], r(2, 4, 50, 64).transpose(1, 2), r(1, 50, 4, 64).expand(2, 50, 4, 64)]
    return t + ([r(2, 9, 2, 4, 64)[:, :, 1], r(2, 9, 4, 64)] if prefix else [])


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("hook", [*HOOKS, "save_on_cpu"])
def test_backward_reads_what_saved_tensor_hooks_return(pkg, told, hook, dtype, prefix):
    """Hooks may return a saved tensor in another layout: the kernels are told the strides of what they are given."""
    tensors = operands(dtype, prefix)
    leaves = [t.detach().requires_grad_(True) for t in tensors]
    lengths, start = torch.tensor([50, 31]), torch.tensor([0, 3], dtype=torch.int32)
    kw = dict(key_lengths=lengths, query_start=start, window=9)
    if prefix:
        kw["prefix_lengths"] = torch.tensor([9, 4], dtype=torch.int32)
    context = torch.autograd.graph.save_on_cpu() if hook == "save_on_cpu" else \
        torch.autograd.graph.saved_tensors_hooks(lambda t: t, HOOKS[hook])
    with context:
        out = (pkg.prefix_attention if prefix else pkg.window_attention)(*leaves, **kw)
    torch.autograd.grad(out, leaves, [torch.ones_like(out)])
    (plan, out, saved, g, given, vectors), = told
    for name, t, want in zip("q k v pk pv".split(), given, tensors):
        assert torch.equal(t, want) and t.dtype == want.dtype and t.data_ptr() % 16 == 0 and t.stride(3) == 1, name
        have = getattr(plan.shape, name + "_strides")
        assert all(n < 2 or a == b for n, a, b in zip(t.shape, have, t.stride())), name
    assert (plan.shape.window, plan.shape.Lq, plan.shape.Lk, plan.shape.groups) == (9, 50, 50, 2 if prefix else 0)
    assert all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in (out, saved, g))
    assert vectors[0].tolist() == [50, 31] and vectors[1].tolist() == [0, 3] and (not prefix or vectors[2].tolist() == [9, 4])
    assert all(v is None or (v.is_contiguous() and v.dtype is torch.int32) for v in vectors)


@pytest.mark.parametrize("at", range(5))
@pytest.mark.parametrize("hook", [lambda t: t.double(), lambda t: t[..., :-1]], ids=["type", "shape"])
def test_backward_refuses_what_is_no_saved_tensor(pkg, told, hook, at):
    """A hook that returns something else than it was given: not read as if it were it. at: of the tensors in the order they are
    unpacked (the vector of lengths, out, the statistics, q, k)."""
    count = iter(range(100))
    leaves = [t.detach().requires_grad_(True) for t in operands(BF, False)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: hook(t) if next(count) == at else t):
        out = pkg.window_attention(*leaves, key_lengths=torch.tensor([50, 31]))
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(out, leaves, [torch.ones_like(out)])
    assert not told


@pytest.mark.parametrize("what", [None, [1.0], 3], ids=["None", "list", "number"])
def test_what_is_no_tensor_is_refused_by_name(pkg, what):
    t = dict(q=heads(), k=heads(), v=heads(), prefix_k=heads(L=9), prefix_v=heads(L=9))
    for fn, names in ((pkg.window_attention, "q k v"), (pkg.prefix_attention, "q k v prefix_k prefix_v")):
        for bad in ([n] for n in names.split()):
            with pytest.raises(RuntimeError, match=f"{bad[0]} must be a tensor, got a {type(what).__name__}"):
                fn(*[what if n in bad else t[n] for n in names.split()])
    for prefix in ((what, what), (t["prefix_k"][0], what)):
        with pytest.raises(RuntimeError, match="prefix_[kv] must be a tensor"):
            pkg.prefix_attention(*list(t.values())[:3], *prefix)
    if what is not None:
        for name in ("key_lengths", "prefix_lengths"):
            with pytest.raises(RuntimeError, match=f"{name} must be a tensor"):
                pkg.prefix_attention(*t.values(), **{name: what})


@pytest.mark.parametrize("name", ["q", "k", "v", "prefix_k", "prefix_v"])
def test_rows_wider_than_the_kernels_take_are_refused(pkg, told, name):
    """A contiguous copy does not help where a token's heads alone are past the limit of token strides."""
    wide, narrow = (torch.zeros(1).expand(1, 2, h, 128) for h in (1 << 15, 1))
    t = dict(q=wide, k=narrow, v=narrow, prefix_k=narrow, prefix_v=narrow)
    if name != "q":
        t = dict(q=wide[:, :1], k=wide[:, :1], v=wide[:, :1], prefix_k=wide[:, :1], prefix_v=wide[:, :1])
        t.update({n: wide for n in (("k", "v") if name in "kv" else ("prefix_k", "prefix_v"))})
    with pytest.raises(RuntimeError, match="heads of a token"):
        pkg.prefix_attention(*t.values())


LAUNCHES = [  # sizes, the forward's and the backward's refusal: fewer than 2^32 work items a launch, whatever the tensors' sizes
    (dict(B=1 << 16, Lq=1, Lk=2, H=12, Hk=12), False, False),      # many samples of one token
    (dict(B=(1 << 20) - 1, Lq=1, Lk=2, H=8, Hk=8), False, False),  # 512 work items for up to 32 rows
    (dict(B=1 << 20, Lq=1, Lk=2, H=8, Hk=8), True, False),
    (dict(B=1, Lq=1 << 28, Lk=1 << 28, H=1, Hk=1, D=8, dtype=0), False, False),
    (dict(B=2, Lq=1 << 28, Lk=1 << 28, H=1, Hk=1, D=8, dtype=0), True, True),
    (dict(B=1 << 13, Lq=1, Lk=1 << 16, H=1, Hk=1, D=8, dtype=0), False, True),  # a backward of many keys, a forward of few rows
]


@pytest.mark.parametrize("case", LAUNCHES, ids=str)
def test_limits_of_a_launch(pkg, case):
    L, lib = pkg._lib, pkg._lib.load()
    kw, fwd, bwd = dict(case[0]), *case[1:]
    if "dtype" in kw:
        kw["dtype"] = L.F32
    D, H = kw.get("D", 64), kw["H"]
    for n, length in (("q", "Lq"), ("k", "Lk"), ("v", "Lk")):
        kw[n] = (kw[length] * H * D, H * D, D)
    s = shape(L, window=16, first=0, **kw)
    need = [lib.mlora_past_attention_workspace_bytes(s), lib.mlora_past_attention_backward_workspace_bytes(s)]
    assert [n == L.ERR_LIMIT for n in need] == [fwd, bwd] and all(n >= 0 or n == L.ERR_LIMIT for n in need)
    ptr = [0x1000] * 3 + [None] * 5
    if fwd:
        assert lib.mlora_past_attention(s, *ptr, 0x2000, 0x3000, 0x4000, 0x5000, 1 << 40, None) == L.ERR_LIMIT
    if bwd:
        assert lib.mlora_past_attention_backward(s, *ptr, 0x2000, 0x3000, 0x4000, 0x6000, (ctypes.c_int64 * 3)(*kw["q"]),
                                                 *[0x7000] * 3, None, None, 0x5000, 1 << 50, None) == L.ERR_LIMIT


def test_a_backward_past_its_limit_does_not_refuse_the_forward(pkg, on_device, monkeypatch):
    monkeypatch.setattr(pkg.kernels, "_call", lambda *a: None)
    q = torch.zeros(1, 1, 1, 8)
    k = torch.zeros(1, 1, 1, 8).expand(1 << 13, 1 << 16, 1, 8)
    q = q.expand(1 << 13, 1, 1, 8)
    assert pkg.window_attention(q, k, k, window=16).shape == q.shape
    with pytest.raises(RuntimeError, match="limit"):
        pkg.window_attention(q.detach().requires_grad_(True), k, k, window=16)


@pytest.mark.parametrize("case", past_plans.PLANS, ids=str)
def test_how_dk_and_dv_are_cut(pkg, case):
    """The calls of the GPU test of the same name are cut as the table says: the shares' sums are what the workspace holds."""
    L, lib = pkg._lib, pkg._lib.load()
    groups, each, n, Lp, H, Hk, window, sinks, chunk = case[:9]
    s = shape(L, B=max(groups, 1) * each, Lq=n, Lk=n, H=H, Hk=Hk, D=128, groups=groups, Lp=Lp, window=window or 0, sinks=sinks, chunk=chunk,
              first=0)
    dq, dkv = past_plans.workspace_bytes(case)
    assert lib.mlora_past_attention_backward_workspace_bytes(s) == max(dq, dkv) and (dq < dkv or max(case[9:]) == case[9])


def test_every_cut_is_in_the_table():
    for waves in (8, 4):
        rows = [c for c in past_plans.PLANS if c[9] == waves]
        assert {(c[11] > 1, c[12] > 1, c[13] > 1) for c in rows} >= {(a, b, c) for a in (0, 1) for b in (0, 1) for c in (0, 1) if a + b < 2} - (
            {(0, 0, 0)} if waves == 4 else set())

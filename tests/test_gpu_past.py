"""Windowed attention with sinks and attention to a shared prefix against the 64-bit definition (past_reference.check derives
the tolerances)."""
import math

import pytest
import torch

import past_plans
import past_reference as ref

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32


def make(dtype, dev, seed, B, Lq, Lk, H, Hk, D, groups=0, Lp=0, loud=1.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, std=1.0: (torch.randn(*s, generator=g) * std).to(dtype).to(dev)  # noqa: E731
    t = [r(B, Lq, H, D, std=loud), r(B, Lk, Hk, D), r(B, Lk, Hk, D)]
    if groups:
        t += [r(groups, Lp, Hk, D), r(groups, Lp, Hk, D)]
    return t, r(B, Lq, H, D)


def run(pkg, tensors, g=None, *, plens=None, lengths=None, start=None, **kw):
    """{"out": ..., "dq": ...} through the public entry points."""
    dev = tensors[0].device
    on = lambda t: t.to(dev) if isinstance(t, torch.Tensor) else t  # noqa: E731
    leaves = [t.detach().requires_grad_(g is not None) for t in tensors]
    if len(tensors) == 3:
        out = pkg.window_attention(*leaves, key_lengths=on(lengths), query_start=on(start), **kw)
    else:
        out = pkg.prefix_attention(*leaves, key_lengths=on(lengths), query_start=on(start), prefix_lengths=on(plens), **kw)
    got = {"out": out.detach()}
    if g is not None:
        got.update(zip(("dq", "dk", "dv", "dpk", "dpv"), torch.autograd.grad(out, leaves, [g])))
    return got


def both(pkg, tensors, g, **kw):
    got = run(pkg, tensors, g, **kw)
    ref.check(got, *tensors, do=g, **kw)
    with torch.no_grad():
        assert torch.equal(run(pkg, tensors, **kw)["out"], got["out"])
    return got


i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731

SEQUENCES = [  # B, L, H, Hk, D, options
    (1, 1, 1, 1, 8, dict(window=1)),
    (2, 2, 2, 1, 16, dict(window=1, sinks=1)),
    (1, 33, 4, 4, 64, dict()),                                   # causal alone
    (2, 64, 4, 2, 40, dict(window=64)),
    (1, 65, 6, 2, 72, dict(window=7, sinks=2)),                  # three heads to a key head: tokens end inside a wave
    (2, 130, 3, 1, 128, dict(window=40, sinks=3, chunk=13)),
    (1, 300, 2, 2, 96, dict(window=128, sinks=70, chunk=64)),    # sinks past a tile
    (1, 517, 5, 1, 64, dict(window=100, sinks=130, chunk=1)),    # sinks and window meet in the first tokens
    (2, 257, 1, 1, 128, dict(window=300, sinks=5, chunk=300)),   # one chunk: everything
    (1, 700, 2, 1, 128, dict(window=33, sinks=1, chunk=32)),
    (1, 1030, 2, 2, 32, dict(window=256, sinks=4)),
]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", SEQUENCES, ids=str)
def test_sequences(pkg, dev, case, ragged, dtype):
    B, L, H, Hk, D, kw = case
    tensors, g = make(dtype, dev, L + H, B, L, L, H, Hk, D)
    lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(L)) if ragged else None
    both(pkg, tensors, g, lengths=lengths, **kw)


CACHES = [  # B, Lq, Lk, H, Hk, D, options
    (3, 1, 700, 8, 2, 128, dict(window=100, sinks=4)),
    (1, 1, 5000, 4, 4, 64, dict(window=4000, sinks=40)),          # shared out and joined
    (2, 5, 333, 6, 2, 72, dict(window=64, sinks=9, chunk=4)),
    (2, 40, 260, 2, 2, 128, dict(window=50, sinks=1)),            # 40 rows: two blocks of rows per wave
    (1, 70, 2100, 4, 2, 96, dict(window=900, sinks=64, chunk=35)),  # more rows than one wave's, shared out
    (2, 156, 999, 3, 3, 128, dict(window=468, sinks=156, chunk=156)),
    (2, 3, 90, 4, 1, 8, dict()),
]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("where", ["end", "lengths", "start", "number"])
@pytest.mark.parametrize("case", CACHES, ids=str)
def test_caches(pkg, dev, case, where, dtype):
    B, Lq, Lk, H, Hk, D, kw = case
    tensors, g = make(dtype, dev, Lk + Lq, B, Lq, Lk, H, Hk, D)
    lengths = i32(*[Lk, Lk // 3, Lq // 2][:B]) if where == "lengths" else None  # fewer keys than queries: padding in front
    start = {"start": i32(*[Lk - 2 * Lq, 0, -1][:B]), "number": Lk // 2}.get(where)
    both(pkg, tensors, g, lengths=lengths, start=start, **kw)


PREFIXES = [  # groups, each, Lq, Lk, Lp, H, Hk, D, options
    (1, 1, 1, 1, 1, 1, 1, 8, dict()),
    (1, 3, 1, 9, 100, 4, 4, 64, dict()),
    (2, 2, 7, 50, 333, 6, 2, 72, dict(window=20)),
    (1, 8, 1, 70, 20000, 8, 8, 128, dict()),                      # computed once for eight samples
    (2, 5, 2, 33, 9001, 8, 4, 128, dict(window=16)),              # 20 rows to a group's key head
    (1, 40, 1, 12, 4100, 8, 2, 128, dict()),                      # 160 rows: the prefix on 128 rows per workgroup
    (3, 2, 65, 65, 130, 2, 1, 128, dict(chunk=65)),
    (1, 2, 200, 200, 515, 3, 3, 40, dict(chunk=50, window=100)),
    (1, 4, 129, 129, 0, 2, 2, 64, dict()),                        # no prefix at all
]


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", PREFIXES, ids=str)
def test_prefixes(pkg, dev, case, ragged, dtype):
    groups, each, Lq, Lk, Lp, H, Hk, D, kw = case
    B = groups * each
    tensors, g = make(dtype, dev, Lp + Lq, B, Lq, Lk, H, Hk, D, groups, Lp)
    gen = torch.Generator().manual_seed(Lp)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen) if ragged else None
    plens = torch.randint(0, Lp + 1, (groups,), generator=gen, dtype=torch.int32) if ragged else None
    both(pkg, tensors, g, lengths=lengths, plens=plens, **kw)
    if groups == 1 and not ragged:  # a prefix without a group axis
        flat = [*tensors[:3], tensors[3][0], tensors[4][0]]
        with torch.no_grad():
            assert torch.equal(pkg.prefix_attention(*flat, **kw), run(pkg, tensors, **kw)["out"])


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq", [1, 40, 150])
def test_what_no_token_sees_may_hold_anything(pkg, dev, Lq, dtype):
    """Keys behind a sample's length, between the sinks and the window of its first token, and behind its last token's chunk;
    padding queries and their upstream gradients: NaN, infinities, the type's lowest value. Samples without a key or whose
    queries are all padding give zeros."""
    B, Lk, H, D = 4, 400, 2, 64
    tensors, g = make(dtype, dev, 5, B, Lq, Lk, H, H, D, 2, 90)
    lengths, plens = i32(400, 390, 0, 300), i32(90, 33)
    start = i32(200, 390 - Lq // 2, 0, -Lq)
    kw = dict(window=60, chunk=4, lengths=lengths, start=start)
    for t, more in ((tensors[:3], dict(sinks=5)), (tensors, dict(plens=plens))):
        got = run(pkg, t, g, **kw, **more)
        ref.check(got, *t, do=g, **kw, **more)
        for name in ("out", "dq", "dk", "dv"):
            assert got[name][2].abs().sum() == 0 and got[name][3].abs().sum() == 0
        dirty, dg = [x.clone() for x in t], g.clone()
        for bad_k, bad_v in ((math.nan, math.inf), (math.inf, math.nan), (torch.finfo(dtype).min, -math.inf)):
            for b, (n, first) in enumerate(ref.starts_of(B, Lq, Lk, lengths, start)):
                vis = ref.seen(Lq, Lk, n, first, 60, more.get("sinks", 0), 4)
                dirty[1][b, ~vis.any(0).to(dev)], dirty[2][b, ~vis.any(0).to(dev)] = bad_k, bad_v
                dirty[0][b, ~vis.any(1).to(dev)], dg[b, ~vis.any(1).to(dev)] = bad_v, bad_k
            if len(t) == 5:
                dirty[3][1, 33:], dirty[4][1, 33:] = bad_k, bad_v
            again = run(pkg, dirty, dg, **kw, **more)
            assert all(torch.equal(got[n], again[n]) for n in got)


def test_int64_vectors_and_values_out_of_range(pkg, dev):
    tensors, g = make(BF, dev, 6, 3, 9, 50, 2, 2, 64, 3, 20)
    for dt in (torch.int32, torch.int64):
        far = 2 ** 31 - 1 if dt is torch.int32 else 2 ** 40
        lengths, plens, start = (torch.tensor(v, dtype=dt) for v in ([-5, far, 17], [far, -1, 3], [41, -far, far]))
        both(pkg, tensors, g, lengths=lengths, plens=plens, start=start, window=8)
        got = both(pkg, tensors, g, start=far)
        assert got["out"].abs().sum() == 0


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq", [2, 100])
def test_options_past_the_range(pkg, dev, Lq, dtype):
    """Windows, chunks and sinks of any size mean all keys; a given scale; loud scores that rise and fall along the keys."""
    tensors, g = make(dtype, dev, 8, 2, Lq, 150, 2, 1, 32, loud=6.0)
    big = 2 ** 40
    whole = both(pkg, tensors, g, scale=0.3)
    for kw in (dict(window=big), dict(window=1, sinks=big)):
        got = run(pkg, tensors, g, scale=0.3, **kw)
        assert torch.equal(got["out"], whole["out"]) or kw.get("window") == 1
        ref.check(got, *tensors, do=g, scale=0.3, **kw)
    ramp = torch.linspace(0.1, 8.0, 150, device=dev).view(1, 150, 1, 1).to(dtype)
    for r in (ramp, ramp.flip(1)):
        both(pkg, [tensors[0], tensors[1] * r, tensors[2]], g, window=big, chunk=big)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq, Lk", [(3, 50), (3, 3000), (200, 200)])
def test_very_low_scores_are_scores(pkg, dev, Lq, Lk, dtype):
    """Every score -2^103 (exact in bf16 and float32): all visible keys weigh the same, forward and backward: dv is the sum of
    do over the rows that see the key, each with weight 1 / its number of keys."""
    (q, k, v), g = make(dtype, dev, 5, 1, Lq, Lk, 2, 2, 32)
    q, k = torch.full_like(q, 2.0 ** 49), torch.full_like(k, -(2.0 ** 49))
    got = run(pkg, [q, k, v], g, window=40, sinks=3, scale=1.0)
    vis = ref.seen(Lq, Lk, Lk, Lk - Lq, 40, 3, 1).double()
    p = vis / vis.sum(1, keepdim=True)
    u = ref.half_step(dtype)
    for name, w, t in (("out", p, v), ("dv", p.T, g)):
        t = ref.f64(t)[0]
        want, size = (torch.einsum("ij,jhd->ihd", w, x) for x in (t, t.abs()))
        room = u * want.abs() + (2 ** -20 + 50 * 2 ** -24 + (u if dtype is BF else 0)) * size
        assert ((ref.f64(got[name])[0] - want).abs() <= room).all(), name


def test_layouts(pkg, dev):
    """q of one packed [B, L, 3, H, D], k and v slices of a joint cache, head-major storage, misaligned storage, token strides
    past the kernels' limit, an expanded batch, a transposed gradient."""
    H, D = 4, 64
    gen = torch.Generator().manual_seed(9)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev).to(BF)  # noqa: E731
    q, kv, g = r(2, 50, 3, H, D)[:, :, 1], r(2, 90, 2, H, D), r(2, H, 50, D).transpose(1, 2)
    both(pkg, [q, kv[:, :, 0], kv[:, :, 1]], g, window=20, sinks=2)
    head_major = r(2, H, 90, D).transpose(1, 2)
    odd = r(2 * 90 * H * D + 3)[3:].view(2, 90, H, D)
    both(pkg, [q, head_major, odd], g, window=20)
    one = r(1, 90, H, D).expand(2, 90, H, D)
    both(pkg, [q, one, kv[:, :, 1], r(1, 40, 2, H, D)[:, :, 1], r(1, H, 40, D).transpose(1, 2)], g, chunk=10)
    wide = r(3, (1 << 22) + 8).as_strided((1, 3, H, D), (0, (1 << 22) + 8, D, 1))
    both(pkg, [wide, wide, wide], torch.ones_like(wide), window=2)


@pytest.mark.parametrize("shape", [(0, 5, 7, 3), (2, 0, 7, 3), (2, 5, 0, 3), (2, 5, 7, 0), (2, 0, 0, 0)])
def test_empty(pkg, dev, shape):
    B, Lq, Lk, Lp = shape
    tensors, g = make(BF, dev, 1, B, Lq, Lk, 4, 2, 64, 1, Lp)
    for t in (tensors[:3], tensors):
        got = run(pkg, t, g, start=0)
        ref.check(got, *t, do=g, start=0)


def test_fixed_order_and_partial_gradients(pkg, dev):
    tensors, g = make(BF, dev, 3, 4, 130, 130, 4, 2, 128, 2, 300)
    first = run(pkg, tensors, g, chunk=10)
    again = run(pkg, tensors, g, chunk=10)
    assert all(torch.equal(first[n], again[n]) for n in first)
    for i, name in enumerate(("dq", "dk", "dv", "dpk", "dpv")):
        leaves = [t.detach().requires_grad_(j == i) for j, t in enumerate(tensors)]
        got, = torch.autograd.grad(pkg.prefix_attention(*leaves, chunk=10), [leaves[i]], [g])
        assert torch.equal(got, first[name])
    x = tensors[0].detach().requires_grad_(True)
    with pytest.raises(RuntimeError):  # the backward itself is not differentiable, and says so
        (d,) = torch.autograd.grad(pkg.window_attention(x, *tensors[1:3]), [x], [g], create_graph=True)
        d.float().sum().backward()


def test_gradient_against_differences(pkg, dev):
    """The kernel's float32 gradients against differences of the 64-bit definition."""
    from block_reference import finite_difference
    tensors, g = make(F, dev, 13, 4, 9, 21, 4, 2, 32, 2, 6)
    kw = dict(window=5, chunk=2, lengths=i32(21, 12, 9, 4), plens=i32(6, 2))
    got = run(pkg, tensors, g, **kw)
    args = [ref.f64(t) for t in tensors]
    for i, name in enumerate(("dq", "dk", "dv", "dpk", "dpv")):
        d = torch.randn(args[i].shape, generator=torch.Generator().manual_seed(i)).double()

        def f(x, i=i):
            return float((ref.attention(*(x if j == i else t for j, t in enumerate(args)), **kw)[0]["out"] * ref.f64(g)).sum())

        want = finite_difference(f, args[i], d, 1e-5)
        have = ref.f64(got[name]) * d
        assert abs(float(have.sum()) - want) <= 2 ** -15 * float(have.abs().sum()) + 1e-6


def test_captured_and_replayed(pkg, dev):
    """Training, a cache's next token and a shared prefix in one HIP graph, replayed with other inputs and lengths."""
    train, g = make(BF, dev, 19, 2, 300, 300, 2, 1, 128)
    token, _ = make(BF, dev, 20, 2, 1, 6000, 4, 2, 128)
    shared, _ = make(BF, dev, 21, 8, 1, 30, 8, 8, 128, 1, 9000)
    lengths = torch.tensor([300, 200], dtype=torch.int32, device=dev)
    filled = torch.tensor([6000, 10], dtype=torch.int32, device=dev)
    for t in train:
        t.requires_grad_(True)

    def step():
        out = pkg.window_attention(*train, window=70, sinks=2, key_lengths=lengths)
        with torch.no_grad():
            more = [pkg.window_attention(*token, window=4000, sinks=4, key_lengths=filled), pkg.prefix_attention(*shared)]
        return [out.detach(), *more, *torch.autograd.grad(out, train, [g])]

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
            for t in (*train, g, *token, *shared):
                t.copy_(torch.randn(t.shape, generator=gen))
            lengths.fill_(90 * seed)
            filled.copy_(torch.tensor([1500 * seed + 1, 5000 - seed]))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_two_streams_at_once(pkg, dev):
    """Calls on two streams have workspaces of their own."""
    a, ga = make(BF, dev, 31, 1, 500, 500, 4, 4, 128)
    b, gb = make(BF, dev, 32, 8, 1, 40, 8, 8, 128, 1, 9000)
    want = run(pkg, a, ga, window=100, sinks=3), run(pkg, b, gb)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(3):
        for s, args, kw in ((streams[0], (a, ga), dict(window=100, sinks=3)), (streams[1], (b, gb), {})):
            with torch.cuda.stream(s):
                got.append(run(pkg, *args, **kw))
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert all(torch.equal(x[n], want[i % 2][n]) for n in x)


def test_a_frame_of_a_long_clip(pkg, dev):
    """A late frame of a Wan clip, tokens and keys of whole frames, two heads of it in 64 bits."""
    L, C, H, D = 12480, 1560, 2, 128
    tensors, _ = make(BF, dev, 23, 1, C, L, H, H, D)
    got = run(pkg, tensors, window=4 * C, sinks=C, chunk=C)
    keys = [*range(C), *range(L - 4 * C, L)]
    q, k, v = (t[:, keys] if t.shape[1] == L else t for t in tensors)
    ref.check(got, q, k, v, chunk=len(keys), start=0)


def test_offsets_past_32_bits(pkg, dev):
    """The last tokens of a cache of 2^31 + elements per sample and a prefix behind 2^31 elements."""
    H, D, Lk = 8, 128, 1100000  # 1.13e9 elements a sample: 4.5 GB for k and v in bf16
    base = torch.zeros(2 * Lk, 2, H, D, dtype=BF, device=dev)
    tail, g = make(BF, dev, 29, 1, 4, 600, H, H, D)
    base[-600:, 0], base[-600:, 1] = tail[1][0], tail[2][0]
    k, v = base[Lk:, 0].unsqueeze(0), base[Lk:, 1].unsqueeze(0)
    got = run(pkg, [tail[0], k, v], window=500, sinks=0)
    ref.check(got, *tail, window=500)
    whole = base.view(1, 2 * Lk, 2, H, D)  # token offsets of 4.5e9 elements
    got = run(pkg, [tail[0], whole[:, :, 0], whole[:, :, 1]], window=500)
    ref.check(got, *tail, window=500)


def some_heads(pkg, tensors, g, heads, **kw):
    """As `both`, for many heads (each with its own key head): those of `heads` against the definition."""
    got = run(pkg, tensors, g, **kw)
    ref.check({n: t[:, :, heads].contiguous() for n, t in got.items()}, *[t[:, :, heads] for t in tensors], do=g[:, :, heads], **kw)
    return got


MANY_BLOCKS = [  # groups, each, L, Lp, H, D, options: more blocks of 256 keys than compute units
    (0, 1, 1100, 0, 64, 128, dict(window=600, sinks=300, chunk=275)),   # sinks in blocks of their own
    (0, 1, 520, 0, 256, 72, dict(chunk=520)),
    (2, 3, 200, 900, 64, 128, dict(window=100)),                        # a prefix that three samples add to
    (0, 2, 1024, 0, 48, 64, dict(window=130, sinks=5)),
]


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", MANY_BLOCKS, ids=str)
def test_many_blocks(pkg, dev, case, ragged):
    groups, each, L, Lp, H, D, kw = case
    B = max(groups, 1) * each
    tensors, g = make(BF, dev, L, B, L, L, H, H, D, groups, Lp)
    gen = torch.Generator().manual_seed(H)
    lengths = torch.randint(0, L + 1, (B,), generator=gen) if ragged else None
    plens = i32(Lp, Lp // 3) if ragged and groups else None
    more = dict(kw, plens=plens) if groups else kw
    some_heads(pkg, tensors, g, [0, H // 2, H - 1], lengths=lengths, **more)


SHARED_OUT = [  # dtype, B, Lq, Lk, H, Hk, D, groups, Lp, options: few rows or heads, so that keys and rows are shared out and joined
    (BF, 1, 2600, 2600, 2, 1, 128, 0, 0, dict(chunk=100)),
    (BF, 3, 700, 700, 4, 2, 128, 1, 900, dict()),
    (BF, 1, 1300, 1300, 4, 2, 96, 0, 0, dict(window=300, sinks=200, chunk=7)),
    (BF, 2, 600, 2000, 2, 2, 64, 0, 0, dict()),
    (F, 1, 40, 3000, 2, 1, 128, 1, 2000, dict()),
    (F, 1, 700, 700, 3, 1, 128, 0, 0, dict(window=90, sinks=130)),
    (F, 2, 260, 1100, 2, 2, 64, 0, 0, dict(chunk=260)),
]


@pytest.mark.parametrize("case", SHARED_OUT, ids=str)
def test_shared_out(pkg, dev, case):
    dtype, B, Lq, Lk, H, Hk, D, groups, Lp, kw = case
    tensors, g = make(dtype, dev, Lq + Lp, B, Lq, Lk, H, Hk, D, groups, Lp)
    got = both(pkg, tensors, g, **kw)
    again = run(pkg, tensors, g, **kw)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("D", [64, 128])
def test_float32_with_many_workgroups(pkg, dev, D):
    """More workgroups of 32 rows than compute units, whose waves are halved."""
    tensors, g = make(F, dev, D, 2, 420, 420, 24, 24, D)
    some_heads(pkg, tensors, g, [0, 11, 23], window=77, sinks=40, lengths=i32(420, 333))


@pytest.mark.parametrize("dtype", [BF, F])
def test_backward_of_gradients_in_any_layout(pkg, dev, dtype):
    """An upstream gradient that is expanded, strided by token, misaligned or of another type."""
    tensors, _ = make(dtype, dev, 41, 2, 70, 70, 4, 2, 64)
    gen = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev).to(dtype)  # noqa: E731
    for g in (r(1, 1, 1, 64).expand(2, 70, 4, 64), r(2, 70, 3, 4, 64)[:, :, 1], r(2 * 70 * 4 * 64 + 1)[1:].view(2, 70, 4, 64)):
        got = run(pkg, tensors, g, window=9)
        same = run(pkg, tensors, g.contiguous().clone(), window=9)
        ref.check(got, *tensors, do=g, window=9)
        assert all(torch.equal(got[n], same[n]) for n in got)


def test_calls_that_follow_each_other(pkg, dev):
    """A streaming sampler and its training pass as they are used together: chunks generated one after the other against a growing
    cache give what the whole sequence gives in one pass, forward, and the gradients of that pass are the definition's."""
    C, n, H, D = 40, 6, 4, 64
    (q, k, v), g = make(BF, dev, 51, 2, C * n, C * n, H, H, D)
    kw = dict(window=2 * C, sinks=C, chunk=C)
    whole = both(pkg, [q, k, v], g, **kw)["out"]
    cache_k, cache_v = torch.full_like(k, math.nan), torch.full_like(v, math.nan)
    u = ref.half_step(BF)
    with torch.no_grad():
        for i in range(n):
            at = slice(i * C, (i + 1) * C)
            cache_k[:, at], cache_v[:, at] = k[:, at], v[:, at]
            filled = torch.full((2,), (i + 1) * C, dtype=torch.int32, device=dev)
            step = pkg.window_attention(q[:, at], cache_k, cache_v, key_lengths=filled, **kw)
            # each within u |out| + 1.3 u (sum p |v| + |out|) of the exact value (past_reference.check), u for the rounding of out and
            # of the weights, 0.3 u for the scores' and sums'; sum p |v| <= max |v|
            room = 6 * u * whole[:, at].float().abs() + 3 * u * v.float().abs().max()
            assert ((step.float() - whole[:, at].float()).abs() <= room).all()
        # both samples' third chunk as continuations of the first one's past
        past = k[:1, :2 * C], v[:1, :2 * C]
        own = slice(2 * C, 3 * C)
        shared = pkg.prefix_attention(q[:, own], k[:, own], v[:, own], past[0][0], past[1][0], chunk=C)
    ref.check({"out": shared}, q[:, own], k[:, own], v[:, own], *past, chunk=C)


def test_float32_between_one_and_two_rounds(pkg, dev):
    """512 to 1024 workgroups of few tiles: a quarter of the waves."""
    tensors, g = make(F, dev, 61, 2, 600, 600, 18, 18, 64)
    some_heads(pkg, tensors, g, [0, 9, 17], window=60, sinks=3, lengths=i32(555, 600))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("prefix", [False, True])
def test_gradients_under_saved_tensor_hooks(pkg, dev, prefix, dtype):
    """Tensors that are offloaded, copied or laid out anew between forward and backward give the gradients that they give as they lie."""
    gen = torch.Generator().manual_seed(71)
    r = lambda *s: torch.randn(*s, generator=gen).to(dev).to(dtype)  # noqa: E731
    packed = r(2, 150, 3, 4, 64)
    tensors, g = [packed[:, :, 0], r(2, 4, 150, 64).transpose(1, 2), r(1, 150, 4, 64).expand(2, 150, 4, 64)], r(2, 150, 4, 64)
    kw = dict(window=40, lengths=i32(150, 97))
    if prefix:
        past = r(1, 70, 2, 4, 64)
        tensors += [past[:, :, 0], past[:, :, 1]]
    want = both(pkg, tensors, g, **kw)
    lay = lambda t: t.permute(*reversed(range(t.dim()))).contiguous().permute(*reversed(range(t.dim())))  # noqa: E731
    graph = torch.autograd.graph
    for hooks in (graph.save_on_cpu(), graph.save_on_cpu(pin_memory=True), graph.saved_tensors_hooks(torch.clone, torch.clone),
                  graph.saved_tensors_hooks(lambda t: t, lambda t: t.clone(memory_format=torch.contiguous_format)),
                  graph.saved_tensors_hooks(lambda t: t, lay)):
        with hooks:
            got = run(pkg, tensors, g, **kw)
        assert all(torch.equal(got[n], want[n]) for n in want)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq, Lk", [(1, 2), (3, 3)])
def test_many_samples(pkg, dev, Lq, Lk, dtype):
    """A million samples' heads of a few tokens, as the pixels of a clip over its frames: some of them against the definition, all of
    them finite and the same as in a batch of their own."""
    B, H, D = 1 << 16, 16, 8
    tensors, g = make(dtype, dev, 83, B, Lq, Lk, H, H, D)
    lengths = torch.randint(0, Lk + 1, (B,), generator=torch.Generator().manual_seed(5))
    got = run(pkg, tensors, g, lengths=lengths, window=2)
    assert all(t.isfinite().all() for t in got.values())
    for at in (0, 31111, B - 3):
        s = slice(at, at + 3)
        part, pg, n = [t[s] for t in tensors], g[s], lengths[s]
        mine = {k: t[s] for k, t in got.items()}
        ref.check(mine, *part, do=pg, lengths=n, window=2)
        alone = run(pkg, part, pg, lengths=n, window=2)
        assert all(torch.equal(mine[k], alone[k]) for k in mine)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("case", past_plans.PLANS, ids=str)
def test_how_dk_and_dv_are_cut(pkg, dev, case, ragged):
    """Every way to cut the keys' blocks and their rows, the first and the last key head with all its query heads."""
    groups, each, L, Lp, H, Hk, window, sinks, chunk = case[:9]
    B, G = max(groups, 1) * each, H // Hk
    tensors, g = make(BF, dev, L + H, B, L, L, H, Hk, 128, groups, Lp)
    gen = torch.Generator().manual_seed(H)
    lengths = torch.randint(L // 2, L + 1, (B,), generator=gen) if ragged else None
    kw = dict(window=window, chunk=chunk, lengths=lengths)
    kw.update(dict(plens=i32(Lp - 1, Lp // 3)[:groups] if ragged else None) if groups else dict(sinks=sinks))
    got = run(pkg, tensors, g, **kw)
    for hk in {0, Hk - 1}:
        pick = lambda t: t[:, :, hk * G:hk * G + G] if t.shape[2] == H and G > 1 else t[:, :, hk:hk + 1]  # noqa: E731, B023
        ref.check({n: pick(t).contiguous() for n, t in got.items()}, *map(pick, tensors), do=pick(g), **kw)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("Lq", [3, 600])
def test_every_operand_past_32_bits(pkg, dev, Lq, dtype):
    """Tokens of q, k, v and a prefix that lie 2^22 - 8 elements apart, the last ones behind 2^31 elements; a second prefix
    behind as many. Forward and every gradient."""
    H, D, n, far = 2, 64, 600, (1 << 22) - 8
    tensors, g = make(dtype, dev, 91, 2, Lq, n, H, H, D, 2, n)
    base = torch.empty(n * far + 8 * H * D * 2, dtype=dtype, device=dev)
    views, at = [], 0
    for t in tensors:
        v = base.as_strided(t.shape, (H * D, far, D, 1), at)
        v.copy_(t)
        views.append(v)
        at += 2 * H * D
    kw = dict(window=70, chunk=3, lengths=i32(n, 555), plens=i32(n, 599))
    got = run(pkg, views, g, **kw)
    ref.check(got, *tensors, do=g, **kw)
    same = run(pkg, tensors, g, **kw)
    assert all(torch.equal(got[k], same[k]) for k in got)
    apart = base.as_strided((2, n, 2, H, D), (n * far - n * 2 * H * D, 2 * H * D, H * D, D, 1))
    apart[:, :, 0], apart[:, :, 1] = tensors[3], tensors[4]
    got = run(pkg, [*tensors[:3], apart[:, :, 0], apart[:, :, 1]], g, **kw)
    assert all(torch.equal(got[k], same[k]) for k in got)


@pytest.mark.parametrize("dtype", [BF, F])
def test_checkpointed(pkg, dev, dtype):
    """Non-reentrant checkpointing forms the saved tensors again in the backward: the same gradients."""
    from torch.utils.checkpoint import checkpoint
    x = make(dtype, dev, 87, 2, 90, 270, 2, 2, 64)[0][1].reshape(2, 90, 3, 128)
    past = make(dtype, dev, 88, 1, 33, 33, 2, 2, 64)[0][1:]

    def block(x, pk, pv):
        q, k, v = (x[:, :, i].view(2, 90, 2, 64) for i in range(3))
        return pkg.prefix_attention(q, k, v, pk, pv, window=25) + pkg.window_attention(q, k, v, window=25, sinks=2)

    leaves = [t.detach().requires_grad_(True) for t in (x, *past)]
    g = torch.randn(2, 90, 2, 64, generator=torch.Generator().manual_seed(2)).to(dev).to(dtype)
    want = torch.autograd.grad(block(*leaves), leaves, [g])
    got = torch.autograd.grad(checkpoint(block, *leaves, use_reentrant=False), leaves, [g])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [BF, F])
def test_smallest_and_largest_scales(pkg, dev, dtype):
    """Scales at the ends of float32 with scores that stay in its range: the mean of what a token sees, or the key of the largest product."""
    # u |out| for out's rounding and u max |v| for the weights', max |v| < 4, 2^-18 for the sums
    (q, k, v), _ = make(dtype, dev, 89, 1, 70, 70, 2, 2, 32)
    assert v.abs().max() < 4
    vis = ref.seen(70, 70, 70, 0, 20, 2, 1).double()
    for scale in (2.0 ** -140, 2.0 ** -126, 2.0 ** -60):
        got = run(pkg, [q, k, v], window=20, sinks=2, scale=scale)["out"]
        want = torch.einsum("ij,jhd->ihd", vis / vis.sum(1, keepdim=True), ref.f64(v)[0])
        assert ((ref.f64(got)[0] - want).abs() <= 2 * ref.half_step(dtype) * 4 + 2 ** -18).all()
    whole = torch.randint(-3, 4, q.shape, generator=torch.Generator().manual_seed(1)).to(dev).to(dtype)
    s = torch.einsum("ihd,jhd->hij", ref.f64(whole)[0], ref.f64(k.sign())[0]).masked_fill(vis == 0, -math.inf)  # whole numbers
    best = (s == s.amax(-1, keepdim=True)).double()
    want = torch.einsum("hij,jhd->ihd", best / best.sum(-1, keepdim=True), ref.f64(v)[0])
    got = run(pkg, [whole, k.sign(), v], window=20, sinks=2, scale=2.0 ** 100)["out"]
    assert ((ref.f64(got)[0] - want).abs() <= 2 * ref.half_step(dtype) * 4 + 2 ** -18).all()


def test_a_hook_that_returns_another_type_or_shape_is_refused(pkg, dev):
    """Of the same strides, bytes and device too: fp16 in place of bf16, fewer samples of more tokens over the same rows."""
    wide = lambda t: t.new_empty(t.numel()).as_strided((t.shape[0] // 2, t.shape[1] * 2, *t.shape[2:]), t.stride())  # noqa: E731
    half = lambda t: t.to(torch.float16)  # noqa: E731
    for at, hook in ((0, half), (2, half), (4, half), (2, wide)):  # of out, the statistics, q, k, v
        count = iter(range(100))
        q, k, v = (torch.zeros(4, 50, 2, 64, dtype=BF, device=dev).requires_grad_(True) for _ in range(3))
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: hook(t) if next(count) == at else t):  # noqa: B023
            out = pkg.window_attention(q, k, v)
        with pytest.raises(RuntimeError, match="saved-tensor hook"):
            torch.autograd.grad(out, [q, k, v], [torch.ones_like(out)])

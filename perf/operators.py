"""The operators of a DiT block between its linears, as cases that can be timed and checked.

Three operators (`case["op"]`):
  rotary   q and k of one attention: an optional RMSNorm (over the whole row as in Wan, or per head),
           then rotary positions with one to three axes (time, height, width)
  cross    attention of q to an encoder's k / v of another length, with ragged key lengths or a key mask
  joint    what joins two sublayers: x' = residual_scale * x + gate * N_post(y), then the norm and the
           modulation that open the next sublayer

Every case is one pass: forward alone where a model samples, forward and every gradient where it trains.
"""
import math

import torch

own = False
DEV = "cuda"
EPS = 1e-6


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def _rotary(name, B, L, grid, H, Hk, D, axes, **more):
    case = dict(name=name, op="rotary", B=B, L=L, grid=grid, H=H, Hk=Hk, D=D, axes=axes, pairing="adjacent",
                norm="row", positions="whole", dtype="bf16", backward=True)
    case.update(more)
    return case


def _cross(name, B, Lq, Lk, H, Hk, D, **more):
    case = dict(name=name, op="cross", B=B, Lq=Lq, Lk=Lk, H=H, Hk=Hk, D=D, lengths="", keep=1.0, dtype="bf16",
                backward=True)
    case.update(more)
    return case


def _joint(name, B, T, W, **more):
    case = dict(name=name, op="joint", B=B, T=T, W=W, stream="f32", dtype="bf16", norm="layer", post="none",
                gate=True, affine="modulated", residual_scale=1.0, backward=True)
    case.update(more)
    return case


def listed():
    return [
        # a streaming sampler's smallest step: one latent frame of 30 x 52 patches of the Wan-1.3B heads
        _rotary("rotary_frame", 1, 1560, "1,30,52", 12, 12, 128, "44,42,42", backward=False),
        # the generator's and the critic's full clips in training, q and k with their row norms
        _rotary("rotary_wan_train", 2, 32760, "21,30,52", 12, 12, 128, "44,42,42"),
        # an image model in float32: two axes, halves paired, norm per head, a padded batch, key heads shared
        _rotary("rotary_image_f32", 2, 4608, "64,65", 24, 8, 64, "32,32", pairing="halves", norm="head", dtype="f32"),
        # one query token per sample to its prompt (a pooled token, a scoring head): latency counts
        _cross("cross_token", 4, 1, 512, 12, 12, 128, lengths="512,77,1,333", backward=False),
        # few query tokens to everything generated so far: the key axis is the long one
        _cross("cross_long_cache", 1, 16, 65520, 24, 8, 128, backward=False),
        # the teacher's conditional and unconditional passes over the text (512 tokens, 126 of them real)
        _cross("cross_wan_text", 2, 32760, 512, 12, 12, 128, lengths="512,126", backward=False),
        # the critic's training pass over the full text context
        _cross("cross_wan_train", 2, 32760, 512, 12, 12, 128),
        # precision='fp32' training of a small model over masked text of an odd length
        _cross("cross_masked_f32", 2, 1560, 77, 12, 12, 64, keep=0.7, dtype="f32"),
        # one streaming frame: the attention branch joins the float32 stream, the next sublayer's input leaves
        _joint("joint_frame", 1, 1560, 1536, backward=False),
        # ... and both roles' full clips in training, with the gate's and the modulation's gradients
        _joint("joint_wan_train", 2, 32760, 1536),
        # a wider block on a bf16 stream, normed before and after, learned norm weights over all samples
        _joint("joint_sandwich_train", 2, 11040, 5120, stream="bf16", norm="rms", post="rms", affine="plain"),
        # the demo network in float32
        _joint("joint_tiny_f32", 2, 256, 256, dtype="f32", affine="plain", gate=False),
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    return max(lo, v // multiple * multiple)


def draw(rng):
    op = rng.choice(("rotary", "cross", "cross", "joint"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    backward = rng.random() < 0.6
    if op == "rotary":
        D = rng.choice((32, 64, 96, 128))
        H = rng.choice((1, 4, 8, 12, 16, 24, 40))
        Hk = rng.choice([h for h in (1, 4, 8, 12, 16, 24, 40) if H % h == 0])
        B = rng.randint(1, 4)
        n = rng.randint(1, 3)
        cuts = sorted(rng.sample(range(1, D // 2), n - 1))
        axes = ",".join(str(2 * (b - a)) for a, b in zip([0, *cuts], [*cuts, D // 2]))
        L = _log_int(rng, 1, min(32760, 2 * 32760 * 12 * 128 // (B * H * D) // (2 if dtype == "f32" else 1)))
        sides, left = [], L
        for _ in range(n):
            sides.append(_log_int(rng, 1, left))
            left //= sides[-1]
        case = _rotary("", B, L, ",".join(map(str, sides)), H, Hk, D, axes,
                       pairing=rng.choice(("adjacent", "halves")), norm=rng.choice(("none", "head", "row")),
                       positions=rng.choice(("whole", "fractional")), dtype=dtype, backward=backward)
    elif op == "cross":
        B, D = rng.randint(1, 4), rng.choice((32, 40, 64, 72, 80, 96, 128, 128))
        H = rng.choice((1, 4, 8, 12, 16, 24, 40))
        Hk = rng.choice((H, H, *[h for h in (1, 4, 8, 12) if H % h == 0]))
        few = rng.random() < 0.4
        # no more products than the largest listed case; float32 runs on a slower unit
        most = 2 * 32760 * 512 * 12 * 128 // (B * H * D) // (16 if dtype == "f32" else 1)
        if few:
            Lk = _log_int(rng, 64, 65520 * 8 * 128 // (B * Hk * D) if B * Hk * D > 1024 else 65520)
            Lq = _log_int(rng, 1, max(1, min(64, most // Lk)))
        else:
            Lk = _log_int(rng, 1, 2048)
            Lq = _log_int(rng, 1, max(1, min(32760, 2 * 32760 * 12 // (B * H), most // Lk)))
        kind = rng.choice(("all", "lengths", "mask"))
        lengths = ",".join(str(rng.randint(0, Lk)) for _ in range(B)) if kind == "lengths" else ""
        case = _cross("", B, Lq, Lk, H, Hk, D, lengths=lengths,
                      keep=round(rng.uniform(0.05, 0.95), 3) if kind == "mask" else 1.0, dtype=dtype,
                      backward=backward)
    else:
        W = rng.choice((_log_int(rng, 64, 8192, 8), 256, 1536, 5120))
        B = rng.randint(1, 4)
        T = _log_int(rng, 1, max(1, min(32760, 2 * 32760 * 1536 // (B * W) // (2 if dtype == "f32" else 1))))
        case = _joint("", B, T, W, stream="f32" if dtype == "f32" else rng.choice(("f32", "bf16")), dtype=dtype,
                      norm=rng.choice(("layer", "rms")), post=rng.choice(("none", "rms", "layer")),
                      gate=rng.random() < 0.7, affine=rng.choice(("modulated", "plain", "none")),
                      residual_scale=rng.choice((1.0, 1.0, 0.5)), backward=backward)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dtype)


def _positions(case, g):
    """[B, L, axes]: the grid's coordinates in row-major order; tokens behind the grid stay at the origin.
    Fractional ones are a clip at another frame rate and size: steps of 1 / 4 to 2 from a start in [0, 16)."""
    B, L, grid = case["B"], case["L"], _ints(case["grid"])
    n = math.prod(grid)
    pos = torch.zeros(B, L, len(grid), dtype=torch.int32, device=DEV)
    pos[:, :n] = torch.cartesian_prod(*(torch.arange(s, dtype=torch.int32, device=DEV) for s in grid)).view(n, len(grid))
    if case["positions"] == "whole":
        first = torch.randint(0, 64, (B, 1, len(grid)), generator=g, device=DEV, dtype=torch.int32)
        pos[:, :n] += first  # a later chunk of the clip
        return pos
    step = torch.rand(B, 1, len(grid), generator=g, device=DEV) * 1.75 + 0.25
    first = torch.rand(B, 1, len(grid), generator=g, device=DEV) * 16
    fractional = torch.zeros(B, L, len(grid), device=DEV)
    fractional[:, :n] = pos[:, :n] * step + first
    return fractional


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]
    if case["op"] == "rotary":
        B, L, H, Hk, D = (case[k] for k in ("B", "L", "H", "Hk", "D"))
        d = dict(q=_randn(g, B, L, H, D, dtype=dt), k=_randn(g, B, L, Hk, D, dtype=dt), positions=_positions(case, g))
        if case["norm"] != "none":  # a trained norm's weights
            d["qw"], d["kw"] = ((1 + _randn(g, h * D if case["norm"] == "row" else D, std=0.1)).to(dt) for h in (H, Hk))
        if case["backward"]:
            d["dq"], d["dk"] = _randn(g, B, L, H, D, dtype=dt), _randn(g, B, L, Hk, D, dtype=dt)
        d["leaves"] = [d[k] for k in ("q", "k", "qw", "kw") if k in d]
    elif case["op"] == "cross":
        B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
        # q and k as their norms leave them, some directions louder: scores of a trained model spread over +-5
        d = dict(q=_randn(g, B, Lq, H, D, std=1.5, dtype=dt), k=_randn(g, B, Lk, Hk, D, dtype=dt),
                 v=_randn(g, B, Lk, Hk, D, dtype=dt), lengths=None, mask=None)
        if case["lengths"]:
            d["lengths"] = torch.tensor(_ints(case["lengths"]), dtype=torch.int32, device=DEV)
        if case["keep"] < 1.0:
            d["mask"] = torch.rand(B, Lk, generator=g, device=DEV) < case["keep"]
        if case["backward"]:
            d["do"] = _randn(g, B, Lq, H, D, dtype=dt)
        d["leaves"] = [d["q"], d["k"], d["v"]]
    else:
        B, T, W = case["B"], case["T"], case["W"]
        st = _DT[case["stream"]]
        d = dict(x=_randn(g, B, T, W, std=2.0, dtype=st), y=_randn(g, B, T, W, dtype=dt))
        vec = torch.float32 if case["stream"] == "f32" else dt  # Wan's modulation is float32, a bf16 model's bf16
        if case["post"] != "none":
            d["post_weight"] = (1 + _randn(g, W, std=0.1)).to(vec)
        if case["gate"]:
            d["gate"] = _randn(g, B, W, std=0.5, dtype=vec)
        if case["affine"] == "modulated":
            d["scale"], d["shift"] = _randn(g, B, W, std=0.2, dtype=vec), _randn(g, B, W, std=0.2, dtype=vec)
        elif case["affine"] == "plain":
            d["scale"], d["shift"] = (1 + _randn(g, W, std=0.1)).to(vec), _randn(g, W, std=0.1, dtype=vec)
        if case["backward"]:
            d["dx1"], d["dout"] = _randn(g, B, T, W, dtype=st), _randn(g, B, T, W, dtype=dt)
        d["leaves"] = [d[k] for k in ("x", "y", "gate", "scale", "shift", "post_weight") if k in d]
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["backward"]:
        for t in d["leaves"]:
            t.requires_grad_(True)
    return dict(case=case, **d)


# ------------------------------------------------------------------ the framework's calls

def _call(state):
    """The operator's outputs, through the framework."""
    from __graft_entry__ import load_package

    pkg = load_package()
    case = state["case"]
    if case["op"] == "rotary":
        return pkg.rotary_axes_qk(state["q"], state["k"], state["positions"], _ints(case["axes"]),
                                  pairing=case["pairing"], q_weight=state.get("qw"), k_weight=state.get("kw"), eps=EPS)
    if case["op"] == "cross":
        return [pkg.cross_attention(state["q"], state["k"], state["v"], key_lengths=state["lengths"],
                                    key_mask=state["mask"])]
    return pkg.gated_residual_norm(state["x"], state["y"], state.get("gate"), state.get("scale"), state.get("shift"),
                                   norm=case["norm"], unit_offset=case["affine"] == "modulated",
                                   post_norm=None if case["post"] == "none" else case["post"],
                                   post_weight=state.get("post_weight"), residual_scale=case["residual_scale"], eps=EPS)


def _upstream(state):
    return [state[k] for k in {"rotary": ("dq", "dk"), "cross": ("do",), "joint": ("dx1", "dout")}[state["case"]["op"]]]


# ------------------------------------------------------------------ plain forms, 32 bits

def _pairs(x, pairing):
    """The two members of every rotated pair, [..., D / 2] each."""
    if pairing == "adjacent":
        return x[..., 0::2], x[..., 1::2]
    h = x.shape[-1] // 2
    return x[..., :h], x[..., h:]


def _join(a, b, pairing):
    return torch.stack((a, b), dim=-1).flatten(-2) if pairing == "adjacent" else torch.cat((a, b), dim=-1)


def _turned(x, cos, sin, pairing):
    a, b = _pairs(x, pairing)
    return _join(a * cos - b * sin, a * sin + b * cos, pairing)


def _angles(case, positions):
    """[B, L, 1, D / 2] in 64 bits: pair i of an axis of d channels turns by position * 10000^(-2 i / d)."""
    axes = torch.tensor(_ints(case["axes"]), device=DEV)
    axis = torch.repeat_interleave(torch.arange(len(axes), device=DEV), axes // 2)
    first = (torch.cumsum(axes // 2, 0) - axes // 2)[axis]
    i = torch.arange(case["D"] // 2, device=DEV) - first
    freq = torch.pow(10000.0, -2.0 * i.double() / axes[axis].double())
    return (positions.double()[..., axis] * freq).unsqueeze(2)


def _rms(x, weight):
    """(x / rms(x), 1 / rms(x)): over the whole row for a weight of the row's width, else over each head."""
    dims = (-2, -1) if weight.numel() == x.shape[-2] * x.shape[-1] else (-1,)
    r = (x.square().mean(dim=dims, keepdim=True) + EPS).rsqrt()
    return x * r, r, dims


def _plain_rotary_one(case, x, weight, cos, sin, g):
    B, L, H, D = x.shape
    xf = x.float()
    if weight is None:
        y = _turned(xf, cos, sin, case["pairing"]).to(x.dtype)
        return [y] if g is None else [y, _turned(g.float(), cos, -sin, case["pairing"]).to(x.dtype)]
    n, r, dims = _rms(xf, weight)
    w = weight.float().view(-1, D)
    y = _turned(n * w, cos, sin, case["pairing"]).to(x.dtype)
    if g is None:
        return [y]
    gn = _turned(g.float(), cos, -sin, case["pairing"])
    dw = (gn * n).sum(dim=(0, 1)).view(-1, w.shape[0], D).sum(dim=0)
    h = gn * w
    dx = (h - n * (h * n).mean(dim=dims, keepdim=True)) * r
    return [y, dx.to(x.dtype), dw.view(-1).to(weight.dtype)]


def _plain_rotary(state):
    case = state["case"]
    angles = _angles(case, state["positions"])
    cos, sin = angles.cos().float(), angles.sin().float()
    a = _plain_rotary_one(case, state["q"], state.get("qw"), cos, sin, state.get("dq"))
    b = _plain_rotary_one(case, state["k"], state.get("kw"), cos, sin, state.get("dk"))
    return [t for pair in zip(a, b) for t in pair]  # y_q, y_k, dq, dk, dqw, dkw


def _live(state):
    """[B, 1, 1, Lk]: the keys a sample has."""
    B, Lk = state["case"]["B"], state["case"]["Lk"]
    live = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
    if state["lengths"] is not None:
        live = torch.arange(Lk, device=DEV) < state["lengths"].unsqueeze(1)
    if state["mask"] is not None:
        live = live & state["mask"]
    return live.view(B, 1, 1, Lk)


def _heads(x, G=1):
    """[B, H * G, L, D] in 32 bits, each head G times."""
    return x.float().transpose(1, 2).repeat_interleave(G, dim=1).contiguous()


def _plain_cross(state):
    case, q = state["case"], state["q"]
    G, scale = case["H"] // case["Hk"], case["D"] ** -0.5
    live = _live(state)
    qh, kh, vh = _heads(q), _heads(state["k"], G), _heads(state["v"], G)
    s = torch.matmul(qh, kh.transpose(-1, -2)).mul_(scale).masked_fill_(~live, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(m.isinf(), torch.zeros_like(m), m)).exp_()  # no key at all: every p is 0
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p, vh)
    out = o.transpose(1, 2).to(q.dtype).contiguous()
    if not case["backward"]:
        return [out]
    do = _heads(state["do"])
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, vh.transpose(-1, -2)).sub_((do * o).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kh)
    dk = torch.matmul(ds.transpose(-1, -2), qh)
    B, Lk, Hk, D = state["k"].shape
    dk, dv = (t.view(B, Hk, G, Lk, D).sum(dim=2).transpose(1, 2).to(q.dtype).contiguous() for t in (dk, dv))
    return [out, dq.transpose(1, 2).to(q.dtype).contiguous(), dk, dv]


def _norm32(u, kind):
    c = u - u.mean(dim=-1, keepdim=True) if kind == "layer" else u
    r = (c.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    return c * r, r


def _norm32_back(h, n, r, kind):
    d = h - n * (h * n).mean(dim=-1, keepdim=True)
    if kind == "layer":
        d = d - h.mean(dim=-1, keepdim=True)
    return d * r


def _row(v):
    """[B or 1, 1, W] in 32 bits."""
    return v.float().view(-1, 1, v.shape[-1])


def _sum_like(t, v):
    """The gradient of a vector per sample ([B, W]) or of all ([W]) from its values at every token."""
    return (t.sum(dim=1) if v.dim() == 2 else t.sum(dim=(0, 1))).to(v.dtype)


def _plain_joint(state):
    case, x, y = state["case"], state["x"], state["y"]
    gate, scale, shift, pw = (state.get(k) for k in ("gate", "scale", "shift", "post_weight"))
    a = case["residual_scale"]
    p = y.float()
    if case["post"] != "none":
        pn, pr = _norm32(p, case["post"])
        p = pn * _row(pw)
    u = a * x.float() + (p if gate is None else p * _row(gate))
    n, r = _norm32(u, case["norm"])
    mult = None if scale is None else _row(scale) + (1.0 if case["affine"] == "modulated" else 0.0)
    out = n if scale is None else n * mult + _row(shift)
    outs = [u.to(x.dtype), out.to(y.dtype)]
    if not case["backward"]:
        return outs
    go = state["dout"].float()
    du = _norm32_back(go if mult is None else go * mult, n, r, case["norm"]) + state["dx1"].float()
    dp = du if gate is None else du * _row(gate)
    dy = dp if pw is None else _norm32_back(dp * _row(pw), pn, pr, case["post"])
    grads = {"x": (a * du).to(x.dtype), "y": dy.to(y.dtype)}
    if gate is not None:
        grads["gate"] = _sum_like(du * p, gate)
    if scale is not None:
        grads["scale"], grads["shift"] = _sum_like(go * n, scale), _sum_like(go, shift)
    if pw is not None:
        grads["post_weight"] = _sum_like(dp * pn, pw)
    return outs + list(grads.values())


def run(state):
    if own:
        case = state["case"]
        with torch.set_grad_enabled(case["backward"]):
            outs = list(_call(state))
        if not case["backward"]:
            return outs
        return [*(t.detach() for t in outs), *torch.autograd.grad(outs, state["leaves"], _upstream(state))]
    with torch.no_grad():
        return {"rotary": _plain_rotary, "cross": _plain_cross, "joint": _plain_joint}[state["case"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "rotary":
        rows = case["B"] * case["L"]
        n = rows * (case["H"] + case["Hk"]) * case["D"]
        pos = rows * len(_ints(case["axes"])) * 4
        # in and out; then the upstream gradient in, the input again where a norm needs it, the gradient out
        more = (3 if case["norm"] != "none" else 2) * n * e + pos if case["backward"] else 0
        return {"bytes": 2 * n * e + pos + more, "flops": n * (10 if case["norm"] != "none" else 4) * (3 if case["backward"] else 1)}
    if case["op"] == "cross":
        B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
        keys = sum(_ints(case["lengths"])) if case["lengths"] else int(B * Lk * case["keep"])
        rows = B * Lq * H * D * e
        nbytes, flops = 2 * rows + 2 * keys * Hk * D * e, 4 * H * Lq * keys * D
        if case["backward"]:
            # q, the output and its gradient in, dq out; k and v in, dk and dv out
            nbytes += 4 * rows + 2 * keys * Hk * D * e + 2 * B * Lk * Hk * D * e
            flops += 10 * H * Lq * keys * D
        return {"bytes": nbytes, "flops": flops}
    n = case["B"] * case["T"] * case["W"]
    es = 4 if case["stream"] == "f32" else 2
    nbytes = n * (2 * es + 2 * e)
    if case["backward"]:
        nbytes += n * (3 * es + 3 * e)
    return {"bytes": nbytes, "flops": n * 12 * (3 if case["backward"] else 1)}


# ------------------------------------------------------------------ 64 bits

def _exact_rotary(case, d):
    axes, B, L, D = _ints(case["axes"]), case["B"], case["L"], case["D"]
    # pair t of the head: which axis, and its frequency
    turn = torch.empty(B, L, D // 2, dtype=torch.complex128, device=DEV)
    t = 0
    for a, width in enumerate(axes):
        for i in range(width // 2):
            phi = d["positions"][:, :, a].double() * 10000.0 ** (-2.0 * i / width)
            turn[:, :, t] = torch.polar(torch.ones_like(phi), phi)
            t += 1
    turn = turn.unsqueeze(2)

    def split(x):
        if case["pairing"] == "adjacent":
            return torch.view_as_complex(x.reshape(*x.shape[:3], D // 2, 2).contiguous())
        return torch.complex(x[..., :D // 2].contiguous(), x[..., D // 2:].contiguous())

    def merge(z):
        return torch.view_as_real(z).reshape(*z.shape[:3], D) if case["pairing"] == "adjacent" else torch.cat((z.real, z.imag), -1)

    ys, dxs, dws = [], [], []
    for x, w, g in (("q", "qw", "dq"), ("k", "kw", "dk")):
        x, w, g = d[x].double(), d.get(w), d.get(g)
        H, rstd, n = x.shape[2], None, x
        if w is not None:
            over = H * D if case["norm"] == "row" else D
            flat = x.reshape(B, L, -1, over)
            rstd = 1 / torch.sqrt((flat * flat).sum(-1, keepdim=True) / over + EPS)
            n = (flat * rstd).reshape(B, L, H, D)
            wide = w.double().reshape(-1, D).expand(H, D)
        ys.append(merge(split(n if w is None else n * wide) * turn))
        if g is None:
            continue
        back = merge(split(g.double()) * turn.conj())
        if w is None:
            dxs.append(back)
            continue
        dw = torch.einsum("blhd,blhd->hd", back, n)
        dws.append(dw.reshape(-1) if case["norm"] == "row" else dw.sum(0))
        hn = (back * wide).reshape(B, L, -1, over)
        nn = n.reshape(B, L, -1, over)
        dxs.append(((hn - nn * (hn * nn).sum(-1, keepdim=True) / over) * rstd).reshape(B, L, H, D))
    return ys + dxs + dws


def _exact_cross(case, d):
    B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
    back = case["backward"]
    new = lambda *s: torch.zeros(*s, dtype=torch.float64, device=DEV)  # noqa: E731
    out, dq, dk, dv = new(B, Lq, H, D), new(B, Lq, H, D), new(B, Lk, Hk, D), new(B, Lk, Hk, D)
    for b in range(B):
        keys = torch.arange(Lk, device=DEV)
        if d["lengths"] is not None:
            keys = keys[:int(d["lengths"][b])]
        if d["mask"] is not None:
            keys = keys[d["mask"][b][keys]]
        if keys.numel() == 0:
            continue
        for h in range(H):
            hk = h // (H // Hk)
            q, k, v = d["q"][b, :, h].double(), d["k"][b, keys, hk].double(), d["v"][b, keys, hk].double()
            p = torch.softmax(q @ k.T / math.sqrt(D), dim=1)
            out[b, :, h] = p @ v
            if not back:
                continue
            do = d["do"][b, :, h].double()
            dv[b, keys, hk] += p.T @ do
            dp = do @ v.T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(D)
            dq[b, :, h] = ds @ k
            dk[b, keys, hk] += ds.T @ q
    return [out, dq, dk, dv] if back else [out]


def _exact_joint(case, d):
    W = case["W"]

    def centred(u, kind):
        c = u - u.sum(-1, keepdim=True) / W if kind == "layer" else u
        return c, torch.sqrt((c * c).sum(-1, keepdim=True) / W + EPS)

    def through(h, c, s, kind):
        """The gradient of c / s given the gradient h of the quotient."""
        d0 = h / s - c * (h * c).sum(-1, keepdim=True) / (W * s ** 3)
        return d0 - d0.sum(-1, keepdim=True) / W if kind == "layer" else d0

    wide = lambda k: d[k].double().reshape(-1, 1, W) if k in d else None  # noqa: E731
    x, y, gate, scale, shift, pw = d["x"].double(), d["y"].double(), *map(wide, ("gate", "scale", "shift", "post_weight"))
    p = y
    if pw is not None:
        pc, ps = centred(y, case["post"])
        p = pc / ps * pw
    u = case["residual_scale"] * x + (p * gate if gate is not None else p)
    c, s = centred(u, case["norm"])
    n = c / s
    m = None if scale is None else (scale + 1 if case["affine"] == "modulated" else scale)
    res = [u, n if m is None else n * m + shift]
    if not case["backward"]:
        return res
    go = d["dout"].double()
    du = d["dx1"].double() + through(go if m is None else go * m, c, s, case["norm"])
    dp = du if gate is None else du * gate
    res += [case["residual_scale"] * du, dp if pw is None else through(dp * pw, pc, ps, case["post"])]
    total = lambda t, k: t.sum(1) if d[k].dim() == 2 else t.sum((0, 1))  # noqa: E731
    if gate is not None:
        res.append(total(du * p, "gate"))
    if m is not None:
        res += [total(go * n, "scale"), total(go, "shift")]
    if pw is not None:
        res.append(total(dp * pc / ps, "post_weight"))
    return res


def exact(case, seed):
    d = _inputs(case, seed)
    return {"rotary": _exact_rotary, "cross": _exact_cross, "joint": _exact_joint}[case["op"]](case, d)

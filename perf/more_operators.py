"""Attention of a stream's tokens to their own past, as cases that can be timed and checked.

Two operators (`case["op"]`):
  window   every token attends to the `window` keys up to the end of its own chunk (chunk 1: token by token; a
           frame's tokens see each other) and to the first `sinks` keys of its sample
  prefix   samples that continue one common past: all of the prefix that a group of samples shares, and the
           sample's own keys under the same rule

Lq = Lk are whole sequences (training, prompts), Lq < Lk the newest tokens of a cache. Every case is one pass:
forward alone where a model samples, forward and every gradient where it trains.
"""
import math

import torch

own = False
DEV = "cuda"


def _ints(text):
    return [int(v) for v in text.split(",")] if text else []


def _window(name, B, Lq, Lk, H, Hk, D, window, sinks, chunk, **more):
    case = dict(name=name, op="window", B=B, Lq=Lq, Lk=Lk, H=H, Hk=Hk, D=D, window=window, sinks=sinks, chunk=chunk,
                lengths="", dtype="bf16", backward=True)
    case.update(more)
    return case


def _prefix(name, groups, each, Lq, Lk, Lp, H, Hk, D, chunk, **more):
    """`groups` prefixes of Lp keys, `each` samples on every one of them; window 0: none."""
    case = dict(name=name, op="prefix", B=groups * each, groups=groups, Lq=Lq, Lk=Lk, Lp=Lp, H=H, Hk=Hk, D=D, window=0,
                sinks=0, chunk=chunk, lengths="", prefix_lengths="", dtype="bf16", backward=True)
    case.update(more)
    return case


def listed():
    return [
        # one new token per sequence against a long cache, ragged: window and sinks are all that is read
        _window("window_token", 4, 1, 65520, 16, 8, 128, 4096, 16, 1, lengths="65520,40001,5000,777", backward=False),
        # the smallest model's next token on a short cache: latency counts
        _window("window_token_small", 1, 1, 777, 12, 12, 64, 256, 4, 1, backward=False),
        # a streaming sampler's next frame of 30 x 52 patches: nine frames back and the first one
        _window("window_frame", 1, 1560, 32760, 12, 12, 128, 14040, 1560, 1560, lengths="20280", backward=False),
        # a prompt of an odd length with shared key heads
        _window("window_prompt", 1, 8191, 8191, 40, 8, 128, 2048, 4, 1, backward=False),
        # the streaming student's training pass over a whole clip of 21 frames
        _window("window_clip_train", 1, 32760, 32760, 12, 12, 128, 14040, 1560, 1560),
        # token sequences in a padded batch, key heads shared
        _window("window_tokens_train", 2, 4096, 4096, 16, 4, 128, 1024, 4, 1, lengths="4096,2777"),
        # precision='fp32' training of a small model at odd sizes
        _window("window_f32_train", 2, 1573, 1573, 6, 6, 64, 257, 3, 1, dtype="f32"),
        # many continuations of one long past, one token each
        _prefix("prefix_token", 1, 32, 1, 1560, 32760, 16, 8, 128, 1,
                lengths=",".join(str(1 + 48 * i) for i in range(32)), backward=False),
        # a few continuations of a short prompt: latency counts
        _prefix("prefix_token_small", 1, 8, 1, 64, 512, 12, 12, 64, 1, backward=False),
        # the next frame of a conditional and an unconditional pass over one history
        _prefix("prefix_frame", 1, 2, 1560, 1560, 14040, 12, 12, 128, 1560, backward=False),
        # training of several rollouts from one history, its gradient summed over them
        _prefix("prefix_rollouts_train", 1, 4, 1560, 1560, 4680, 12, 12, 128, 1560),
        # two histories of different lengths in float32, odd sizes, key heads shared
        _prefix("prefix_f32_train", 2, 3, 131, 131, 515, 8, 2, 64, 1, prefix_lengths="515,130", dtype="f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    op = rng.choice(("window", "window", "prefix"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    D = rng.choice((32, 64, 72, 96, 128, 128))
    H = rng.choice((1, 4, 8, 12, 16, 40))
    Hk = rng.choice((H, H, *[h for h in (1, 4, 8) if H % h == 0]))
    cached = rng.random() < 0.45
    # scores of the plain form, and products, within those of the largest listed case; float32 runs on a slower unit
    most = 4_000_000_000 // (16 if dtype == "f32" else 1) // H
    chunk = rng.choice((1, 1, 1, _log_int(rng, 2, 1560)))
    if op == "window":
        B = rng.randint(1, 4)
        if cached:
            Lq = rng.choice((1, 1, _log_int(rng, 2, 64), chunk))
            Lk = _log_int(rng, max(64, Lq), max(64, Lq, min(65520, most // (B * Lq), 65520 * 4096 // (B * Hk * D))))
        else:
            Lk = Lq = _log_int(rng, 64, min(8192, int(math.sqrt(most / B))))
        ragged = rng.random() < 0.5
        lengths = ",".join(str(rng.randint(min(Lk, 8), Lk)) for _ in range(B)) if ragged else ""
        window = max(chunk, _log_int(rng, 16, max(16, 2 * Lk)))
        sinks = rng.choice((0, 1, 4, rng.randint(0, 64), min(chunk, Lk), _log_int(rng, 1, Lk)))
        case = _window("", B, Lq, Lk, H, Hk, D, window, sinks, chunk, lengths=lengths, dtype=dtype,
                       backward=not cached and rng.random() < 0.7)
    else:
        groups, each = rng.choice((1, 1, 2, 3)), _log_int(rng, 1, 32)
        B = groups * each
        room = most // B
        Lq = rng.choice((1, 1, rng.randint(2, 16))) if cached else _log_int(rng, 32, 1560)
        Lp = _log_int(rng, 16, max(16, min(32760, room // Lq // 2, 65520 * 4096 // (B * Hk * D))))
        Lq = min(Lq, max(1, room // (2 * Lp)))
        Lk = _log_int(rng, Lq, max(Lq, 1560)) if cached else Lq
        lengths = ",".join(str(rng.randint(1, Lk)) for _ in range(B)) if rng.random() < 0.5 else ""
        plens = ",".join(str(rng.randint(0, Lp)) for _ in range(groups)) if rng.random() < 0.4 else ""
        case = _prefix("", groups, each, Lq, Lk, Lp, H, Hk, D, chunk, lengths=lengths, prefix_lengths=plens, dtype=dtype,
                       window=rng.choice((0, 0, max(chunk, _log_int(rng, 16, max(16, 2 * Lk))))),
                       backward=not cached and Lq >= 32 and rng.random() < 0.7)
    del case["name"]
    return case


# ------------------------------------------------------------------ inputs

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = _DT[case["dtype"]]
    B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))

    def randn(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEV).mul_(std).to(dt)

    # q and k as their norms leave them, some directions louder: scores of a trained model spread over +-5
    d = dict(q=randn(B, Lq, H, D, std=1.5), k=randn(B, Lk, Hk, D), v=randn(B, Lk, Hk, D), lengths=None, plens=None)
    if case["op"] == "prefix":
        d["pk"], d["pv"] = randn(case["groups"], case["Lp"], Hk, D), randn(case["groups"], case["Lp"], Hk, D)
        if case["prefix_lengths"]:
            d["plens"] = torch.tensor(_ints(case["prefix_lengths"]), dtype=torch.int32, device=DEV)
    if case["lengths"]:
        d["lengths"] = torch.tensor(_ints(case["lengths"]), dtype=torch.int32, device=DEV)
    if case["backward"]:
        d["do"] = randn(B, Lq, H, D)
    d["leaves"] = [d[k] for k in ("q", "k", "v", "pk", "pv") if k in d]
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    if case["backward"]:
        for t in d["leaves"]:
            t.requires_grad_(True)
    return dict(case=case, **d)


# ------------------------------------------------------------------ the framework's calls

def _call(state):
    """The operator's output, through the framework."""
    from __graft_entry__ import load_package

    pkg = load_package()
    case = state["case"]
    if case["op"] == "window":
        return pkg.window_attention(state["q"], state["k"], state["v"], window=case["window"], sinks=case["sinks"],
                                    chunk=case["chunk"], key_lengths=state["lengths"])
    return pkg.prefix_attention(state["q"], state["k"], state["v"], state["pk"], state["pv"], window=case["window"] or None,
                                chunk=case["chunk"], key_lengths=state["lengths"], prefix_lengths=state["plens"])


# ------------------------------------------------------------------ plain form, 32 bits

def _visible(state):
    """[B, 1, 1, Lq, Lp + Lk]: which keys a query has, the prefix's first."""
    case = state["case"]
    B, Lq, Lk, C = case["B"], case["Lq"], case["Lk"], case["chunk"]
    n = state["lengths"]
    n = torch.full((B, 1, 1), Lk, device=DEV) if n is None else n.view(B, 1, 1)
    j = torch.arange(Lk, device=DEV)
    p = torch.arange(Lq, device=DEV).view(1, Lq, 1)
    if Lq < Lk:
        p = p + n - Lq  # the newest tokens of the cache
    token = (p >= 0) & (p < n)
    end = (p // C + 1) * C
    vis = token & (j < torch.minimum(end, n))
    if case["window"]:
        vis &= (j >= end - case["window"]) | (j < case["sinks"])
    if case["op"] == "prefix":
        Lp, each = case["Lp"], B // case["groups"]
        m = state["plens"]
        m = torch.full((B, 1, 1), Lp, device=DEV) if m is None else m.repeat_interleave(each).view(B, 1, 1)
        vis = torch.cat(((torch.arange(Lp, device=DEV) < m) & token.expand(B, Lq, 1), vis.expand(B, Lq, Lk)), dim=-1)
    return vis.expand(B, Lq, vis.shape[-1]).unsqueeze(1).unsqueeze(1)


def _keys(state, name):
    """[B, Hk, 1, keys, D] in 32 bits, the prefix's first."""
    t = state[name].float()
    if state["case"]["op"] == "prefix":
        p = state["p" + name].float()
        t = torch.cat((p.repeat_interleave(t.shape[0] // p.shape[0], dim=0), t), dim=1)
    return t.transpose(1, 2).unsqueeze(2).contiguous()


def _queries(t, Hk):
    """[B, Hk, G, L, D] in 32 bits."""
    B, L, H, D = t.shape
    return t.float().view(B, L, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).contiguous()


def _tokens(t, dtype):
    B, Hk, G, L, D = t.shape
    return t.permute(0, 3, 1, 2, 4).reshape(B, L, Hk * G, D).to(dtype)


def _flat(t):
    """The heads that share keys as rows of one matrix."""
    return t.flatten(2, 3)


def _plain(state):
    case, q = state["case"], state["q"]
    B, Lq, H, D = q.shape
    Hk, scale = case["Hk"], D ** -0.5
    G = H // Hk
    vis = _visible(state)
    n = vis.shape[-1]
    qh, kh, vh = _flat(_queries(q, Hk)), _flat(_keys(state, "k")), _flat(_keys(state, "v"))
    s = torch.matmul(qh, kh.transpose(-1, -2)).mul_(scale)
    s.view(B, Hk, G, Lq, n).masked_fill_(~vis, -math.inf)
    m = s.amax(dim=-1, keepdim=True)
    p = s.sub_(torch.where(m.isinf(), torch.zeros_like(m), m)).exp_()  # no key at all: every p is 0
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    o = torch.matmul(p, vh)
    out = _tokens(o.view(B, Hk, G, Lq, D), q.dtype)
    if not case["backward"]:
        return [out]
    do = _flat(_queries(state["do"], Hk))
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, vh.transpose(-1, -2)).sub_((do * o).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, kh)
    dk = torch.matmul(ds.transpose(-1, -2), qh)
    dq = _tokens(dq.view(B, Hk, G, Lq, D), q.dtype)
    dk, dv = dk.transpose(1, 2), dv.transpose(1, 2)  # [B, keys, Hk, D]
    Lp = n - case["Lk"]
    mine = [t[:, Lp:].to(q.dtype).contiguous() for t in (dk, dv)]
    if case["op"] == "window":
        return [out, dq, *mine]
    shared = [t[:, :Lp].unflatten(0, (case["groups"], -1)).sum(dim=1).to(q.dtype) for t in (dk, dv)]
    return [out, dq, *mine, *shared]


def run(state):
    if own:
        case = state["case"]
        with torch.set_grad_enabled(case["backward"]):
            out = _call(state)
        if not case["backward"]:
            return [out]
        return [out.detach(), *torch.autograd.grad([out], state["leaves"], [state["do"]])]
    with torch.no_grad():
        return _plain(state)


# ------------------------------------------------------------------ what a pass cannot do without

def _sample(case, b):
    """(pairs of query and own key, own keys that some query sees, prefix keys) of sample b."""
    Lq, Lk, C, S = case["Lq"], case["Lk"], case["chunk"], case["sinks"]
    n = _ints(case["lengths"])[b] if case["lengths"] else Lk
    W = case["window"] or Lk + C
    first = n - Lq if Lq < Lk else 0
    pairs, lowest, highest, sinks, p, queries = 0, Lk, 0, 0, max(first, 0), 0
    while p < min(first + Lq, n):  # chunk by chunk
        end = (p // C + 1) * C
        rows = min(end, first + Lq, n) - p
        hi, lo = min(end, n), max(0, end - W)
        extra = min(S, lo, hi)
        pairs += rows * (max(hi - lo, 0) + extra)
        lowest, highest, sinks, queries = min(lowest, lo), max(highest, hi), max(sinks, extra), queries + rows
        p += rows
    prefix = 0
    if case["op"] == "prefix" and queries:
        lens = _ints(case["prefix_lengths"])
        prefix = lens[b * case["groups"] // case["B"]] if lens else case["Lp"]
    return pairs + queries * prefix, max(highest - lowest, 0) + min(sinks, lowest), prefix


def work(case):
    B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
    e = 4 if case["dtype"] == "f32" else 2
    per = [_sample(case, b) for b in range(B)]
    pairs, keys = sum(p[0] for p in per), sum(p[1] for p in per)
    held = B * Lk
    if case["op"] == "prefix":
        each = B // case["groups"]
        keys += sum(max(p[2] for p in per[g * each:(g + 1) * each]) for g in range(case["groups"]))
        held += case["groups"] * case["Lp"]
    rows = B * Lq * H * D * e
    nbytes, flops = 2 * rows + 2 * keys * Hk * D * e, 4 * H * D * pairs
    if case["backward"]:
        # q, the output and its gradient in, dq out; k and v in, dk and dv out
        nbytes += 4 * rows + 2 * keys * Hk * D * e + 2 * held * Hk * D * e
        flops += 10 * H * D * pairs
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    d = _inputs(case, seed)
    B, Lq, Lk, H, Hk, D = (case[k] for k in ("B", "Lq", "Lk", "H", "Hk", "D"))
    back, shared = case["backward"], case["op"] == "prefix"
    new = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=DEV)  # noqa: E731
    out, dq, dk, dv = new(d["q"]), new(d["q"]), new(d["k"]), new(d["v"])
    dpk, dpv = (new(d["pk"]), new(d["pv"])) if shared else (None, None)
    for b in range(B):
        count = int(d["lengths"][b]) if d["lengths"] is not None else Lk
        place = torch.arange(Lq, device=DEV) + (count - Lq if Lq < Lk else 0)
        rows = ((place >= 0) & (place < count)).nonzero().flatten()
        if rows.numel() == 0:
            continue
        block = torch.div(place[rows], case["chunk"], rounding_mode="floor").unsqueeze(1)
        # the own keys from the first that any of these tokens sees, and the sinks before it
        lowest = 0
        if case["window"]:
            lowest = max(0, (int(block[0]) + 1) * case["chunk"] - case["window"])
        keys = torch.cat((torch.arange(min(case["sinks"], lowest), device=DEV), torch.arange(lowest, count, device=DEV)))
        seen = torch.div(keys, case["chunk"], rounding_mode="floor") <= block
        if case["window"]:
            behind = (block + 1) * case["chunk"] - keys  # 1: the last key of the token's chunk
            seen &= (behind <= case["window"]) | (keys < case["sinks"])
        g = b * case["groups"] // B if shared else 0
        m = 0
        if shared:
            m = int(d["plens"][g]) if d["plens"] is not None else case["Lp"]
            seen = torch.cat((torch.ones(rows.numel(), m, dtype=torch.bool, device=DEV), seen), dim=1)
        for h in range(H):
            hk = h // (H // Hk)
            q, k, v = d["q"][b, rows, h].double(), d["k"][b, keys, hk].double(), d["v"][b, keys, hk].double()
            if shared:
                k, v = torch.cat((d["pk"][g, :m, hk].double(), k)), torch.cat((d["pv"][g, :m, hk].double(), v))
            p = torch.softmax((q @ k.T / math.sqrt(D)).masked_fill_(~seen, -math.inf), dim=1)
            out[b, rows, h] = p @ v
            if not back:
                continue
            do = d["do"][b, rows, h].double()
            gv = p.T @ do
            dp = do @ v.T
            dp -= (p * dp).sum(1, keepdim=True)
            ds = dp.mul_(p).div_(math.sqrt(D))
            dq[b, rows, h] = ds @ k
            gk = ds.T @ q
            dk[b, keys, hk] += gk[m:]
            dv[b, keys, hk] += gv[m:]
            if shared:
                dpk[g, :m, hk] += gk[:m]
                dpv[g, :m, hk] += gv[:m]
    if not back:
        return [out]
    return [out, dq, dk, dv, dpk, dpv] if shared else [out, dq, dk, dv]

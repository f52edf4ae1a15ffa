"""Timing cases of the transformer-layer operators on one MI355X: RMS norm with
the residual's addition, rotary positions, and attention over packed sequences
and over a cache.

`listed()` holds the calls that stand for their uses, `draw()` further sizes of
the same ranges.  `run()` computes the operators in elementary torch operations
in 32 bits (angles in 64), or, where `own` is true, by the calls that a program
makes of this framework.  `exact()` restates each definition in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TDT = {"f32": torch.float32, "bf16": torch.bfloat16}
ES = {"f32": 4, "bf16": 2}
EPS = 1e-6
TAIL = 3        # rows behind the last sequence: a program's buffers are longer than what one call fills

_ctx = None


def _vrs():
    """The package, its context made once as a program does."""
    global _ctx
    sys.path[:0] = [] if os.path.join(ROOT, "vision-rs_amd") in sys.path else [os.path.join(ROOT, "vision-rs_amd")]
    import vrs
    if _ctx is None:
        torch.cuda.init()
        _ctx = vrs.Context(0)
    return vrs


# ---- the cases ----------------------------------------------------------------


def _attention(name, dtype, heads, kv, dim, causal, n, q, past, cap, mix):
    return {"name": name, "kind": "attention", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "causal": causal,
            "n": n, "q_lo": q[0], "q_hi": q[1], "past_lo": past[0], "past_hi": past[1], "cap": cap, "mix": mix}


def _norm(name, dtype, rows, cols, res, out):
    return {"name": name, "kind": "norm", "dtype": dtype, "rows": rows, "cols": cols, "res": res, "out": out}


def _rope(name, dtype, heads, kv, dim, rot, layout, axes, scaled, n, q, past, cap, mix):
    return {"name": name, "kind": "rope", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "rot": rot,
            "layout": layout, "axes": axes, "scaled": scaled, "n": n, "q_lo": q[0], "q_hi": q[1],
            "past_lo": past[0], "past_hi": past[1], "cap": cap, "mix": mix}


def listed():
    return [
        # one long prompt through a decoder layer with grouped heads: the largest call, bound by the matrix cores
        _attention("attention-prompt-8192", "bf16", 32, 8, 128, True, 1, (8192, 8192), (0, 0), 0, 1),
        # a batch of prompts of different lengths, packed
        _attention("attention-prompts-packed", "bf16", 32, 8, 128, True, 9, (33, 2800), (0, 0), 0, 2),
        # a batch of images of different sizes through an image encoder: every patch sees every patch of its image
        _attention("attention-images-packed", "bf16", 12, 12, 64, False, 24, (196, 1600), (0, 0), 0, 3),
        # two images of 37 x 37 patches in float32, where results have to agree with a float32 program
        _attention("attention-images-f32", "f32", 6, 6, 64, False, 2, (1369, 1369), (0, 0), 0, 4),
        # the next pieces of four long prompts over what the cache holds of them
        _attention("attention-chunk-cache", "bf16", 32, 8, 128, True, 4, (100, 300), (2000, 9000), 9472, 5),
        # one token of one short conversation: the smallest call, latency
        _attention("attention-token-1", "bf16", 16, 2, 128, True, 1, (1, 1), (700, 700), 1024, 6),
        # one token of each of 64 requests over their caches: bound by memory
        _attention("attention-tokens-64", "bf16", 32, 8, 128, True, 64, (1, 1), (500, 8000), 8192, 7),
        # the norm before a layer, over a long prompt
        _norm("norm-prompt", "bf16", 8192, 4096, True, "same"),
        # the same before an e4m3 product, for the tokens of a few requests: latency
        _norm("norm-tokens-e4m3", "bf16", 8, 4096, True, "group128"),
        # float32, a width that no vector divides, no residual
        _norm("norm-f32-odd", "f32", 1037, 1001, False, "same"),
        # rotary positions of five prompts, keys and values into the cache, frequencies scaled for long contexts
        _rope("rope-prompts-cache", "bf16", 32, 8, 128, 128, "half", 1, True, 5, (400, 3000), (0, 2000), 5120, 8),
        # rows and columns of image patches as two axes, in float32, interleaved pairs
        _rope("rope-images-2d-f32", "f32", 16, 16, 80, 80, "pairs", 2, False, 2, (1369, 1369), (0, 0), 0, 9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    mix = rng.randrange(1 << 20)
    dtype = "bf16" if rng.random() < 0.75 else "f32"
    use = rng.choice(["prompt", "images", "chunk", "tokens", "norm", "rope"])
    if use == "norm":
        cols = _log(rng, 64, 16384)
        out = rng.choice(["same", "same", "row", "group32", "group64", "group128", "step"])
        if out != "same" or rng.random() < 0.5:
            cols = max(128, cols // 128 * 128)     # hidden sizes are mostly such; e4m3 groups divide them
        rows = max(1, min(_log(rng, 1, 20000), (8192 * 4096) // cols))
        c = _norm("", dtype, rows, cols, rng.random() < 0.7, out)
    elif use == "rope":
        dim = rng.choice([32, 64, 80, 96, 128])
        kv = rng.choice([1, 2, 4, 8])
        cached = rng.random() < 0.6
        axes = 1 if cached else rng.choice([1, 2, 3])
        rot = dim if rng.random() < 0.6 else dim // 2
        n = _log(rng, 1, 32)
        hi = max(1, min(_log(rng, 1, 4000), 12000 // n))
        past = _log(rng, 1, 2000) if cached else 0
        c = _rope("", dtype, kv * rng.choice([1, 2, 4]), kv, dim, rot, rng.choice(["half", "pairs"]), axes,
                  rng.random() < 0.5, n, (max(1, hi // rng.choice([1, 2, 7])), hi), (0, past),
                  hi + past + 5 if cached else 0, mix)
    else:
        dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 5, 8] if dtype == "bf16" else [1, 2, 4])
        if use in ("prompt", "images"):
            n = _log(rng, 1, 48)
            # the scores of all sequences at the longest one's size stay below those of the largest listed case
            hi = min(8192 if dtype == "bf16" else 3500, int(math.sqrt(32 * 8192 * 8192 / 2 / (n * heads))))
            hi = _log(rng, 16, hi)
            c = _attention("", dtype, heads, kv, dim, use == "prompt", n, (max(1, hi // rng.choice([1, 2, 9])), hi),
                           (0, 0), 0, mix)
        elif use == "chunk":
            n, past = _log(rng, 1, 8), _log(rng, 50, 8000)
            hi = min(_log(rng, 2, 500), 32 * 8192 * 8192 // 2 // (n * heads * (past + 500)))
            c = _attention("", dtype, heads, kv, dim, True, n, (max(1, hi // rng.choice([1, 3])), hi),
                           (past // rng.choice([1, 2, 5]), past), hi + past + 1, mix)
        else:
            n = _log(rng, 1, 96)
            # no more bytes than the largest listed cache
            past = min(_log(rng, 1, 8000), 64 * 4200 * 8 * 128 * 2 // (n * kv * dim * ES[dtype]))
            q = rng.choice([1, 1, 1, 2, 5])
            c = _attention("", dtype, heads, kv, dim, True, n, (1, q), (past // rng.choice([1, 2, 5]), past),
                           past + q + 7, mix)
    del c["name"]
    return c


def _lengths(case):
    """Queries and earlier keys of each sequence, as a program's scheduler knows them."""
    r = random.Random(case["mix"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(case["n"])]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in range(case["n"])]
    return q, past if case["cap"] else [0] * case["n"]


def work(case):
    es = ES[case["dtype"]]
    if case["kind"] == "norm":
        e = case["rows"] * case["cols"]
        out = es if case["out"] == "same" else 1
        scales = {"row": case["rows"], "group32": e // 32, "group64": e // 64, "group128": e // 128}.get(case["out"], 0)
        return {"bytes": e * (es * (3 if case["res"] else 1) + out) + 4 * case["cols"] + 4 * scales, "flops": 5 * e}
    q, past = _lengths(case)
    if case["kind"] == "rope":
        rows = sum(q)
        e = rows * case["dim"] * (case["heads"] + (2 if case["cap"] else 1) * case["kv"])
        return {"bytes": 2 * e * es + 4 * rows * case["axes"],
                "flops": 3 * rows * case["rot"] * (case["heads"] + case["kv"])}
    pairs = sum(a * (p + a) - (a * (a - 1) // 2 if case["causal"] else 0) for a, p in zip(q, past))
    rows, keys = sum(q), sum(q) + sum(past)
    return {"bytes": es * case["dim"] * (2 * rows * case["heads"] + 2 * keys * case["kv"]),
            "flops": 4 * case["dim"] * case["heads"] * pairs}


# ---- inputs ---------------------------------------------------------------------


def _frequencies(case):
    """Revolutions per position of each pair, in 64 bits: base^(-2 i / pairs of the axis) / 2 pi; scaled: slow pairs
    (under 1 turn over 4096 positions) turn 8 times slower, fast ones (over 4 turns) as before, a ramp between."""
    pairs = case["rot"] // 2
    at = torch.tensor([(i - lo) / (hi - lo) for lo, hi in _axes(case) for i in range(lo, hi)], dtype=torch.float64)
    f = 10000.0 ** -at / (2 * math.pi)
    if case["scaled"]:
        keep = ((f * 4096 - 1.0) / 3.0).clamp(0, 1)
        f = f * keep + f / 8 * (1 - keep)
    assert f.numel() == pairs
    return f


def _axes(case):
    """The pairs of each axis."""
    pairs, a = case["rot"] // 2, case["axes"]
    cut = [pairs * i // a for i in range(a + 1)]
    return list(zip(cut[:-1], cut[1:]))


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TDT[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dt)

    st = {"case": case}
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # activations of a residual stream: a few channels far larger than the rest
        spread = torch.exp(torch.randn(cols, generator=g, device=DEV))
        st["x"] = (torch.randn(rows, cols, generator=g, device=DEV) * spread).to(dt)
        st["res"] = normal(rows, cols) if case["res"] else None
        st["weight"] = 1 + 0.2 * torch.randn(cols, generator=g, device=DEV)
        st["step"] = 1 / 32
        return st
    q, past = _lengths(case)
    k_len = [a + b for a, b in zip(q, past)]
    rows = sum(q) + TAIL
    H, KV, D, cap = case["heads"], case["kv"], case["dim"], case["cap"]
    starts = [sum(q[:i]) for i in range(case["n"] + 1)]
    st["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    # a cache holds the sequences at fixed places; otherwise keys lie at their queries' rows
    st["k_start"] = torch.tensor([i * cap for i in range(case["n"])] if cap else starts[:-1], dtype=torch.int32, device=DEV)
    st["k_len"] = torch.tensor(k_len, dtype=torch.int32, device=DEV)
    st["rows"], st["max_q"], st["max_k"] = sum(q), max(q), max(k_len)
    k_rows = case["n"] * cap if cap else rows
    if case["kind"] == "attention":
        st["q"] = normal(rows, H, D, scale=2.0)      # scores with some weight on single keys
        st["k"], st["v"] = normal(k_rows, KV, D), normal(k_rows, KV, D)
        st["out"] = torch.full((rows, H, D), 1 / 64, dtype=dt, device=DEV)
    else:
        # queries, keys and values as one product leaves them, in one row
        st["qkv"] = normal(rows, (H + 2 * KV), D)
        st["freq"] = _frequencies(case).to(DEV)
        st["q_out"] = torch.full((rows, H, D), 1 / 64, dtype=dt, device=DEV)
        st["k_out"], st["v_out"] = normal(k_rows, KV, D), normal(k_rows, KV, D)
        if case["axes"] > 1:     # rows and columns (and frames) of the patches
            r = torch.arange(rows, device=DEV, dtype=torch.int32)
            st["positions"] = torch.stack([(r // 37 ** i) % 37 for i in range(case["axes"])])
    if own:      # the plan of the batch, which a program makes once and uses in every layer
        vrs = _vrs()
        at_cache = bool(cap)
        st["seqs"] = vrs.seqs(st["q_start"], st["k_start"] if at_cache else None, st["k_len"] if at_cache else None,
                              max_q=st["max_q"], max_k=st["max_k"])
    return st


# ---- the operators ----------------------------------------------------------------


def run(st):
    return {"norm": _run_norm, "rope": _run_rope, "attention": _run_attention}[st["case"]["kind"]](st)


def _run_norm(st):
    c = st["case"]
    out, step = c["out"], st["step"]
    group = {"same": 0, "step": 0, "row": c["cols"]}.get(out) if not out.startswith("group") else int(out[5:])
    if own:
        r = _vrs_norm(st, out, group, step)
        return {k: v.view(torch.float8_e4m3fn) if v.dtype == torch.uint8 else v for k, v in r.items()}
    s = st["x"].float()
    if st["res"] is not None:
        s = s + st["res"].float()
    y = s * torch.rsqrt((s * s).mean(1, keepdim=True) + EPS) * st["weight"]
    r = {"sum": s.to(st["x"].dtype)} if st["res"] is not None else {}
    if out == "same":
        return {"y": y.to(st["x"].dtype), **r}
    if out == "step":
        return {"y": (y / step).clamp(-448, 448).to(torch.float8_e4m3fn), **r}
    g = y.view(y.shape[0], -1, group)
    amax = g.abs().amax(2, keepdim=True)
    scale = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
    return {"y": (g / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(y.shape), "scales": scale.squeeze(2), **r}


def _vrs_norm(st, out, group, step):
    vrs = _vrs()
    res = st["res"]
    y, s, scales = _ctx.rms_norm(st["x"], st["weight"], EPS, res=res, e4m3=out != "same", group=group,
                                 out_step=step if out == "step" else 0.0)
    r = {"y": y}
    if s is not None:
        r["sum"] = s
    if scales is not None:
        r["scales"] = scales
    return r


def _rows(st):
    """Sequence and place in it of each query row."""
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(st["q_start"][1:].long(), row, right=True)
    return seq, row - st["q_start"][seq].long()


def _run_rope(st):
    c = st["case"]
    H, KV, rot = c["heads"], c["kv"], c["rot"]
    q, k, v = st["qkv"][:, :H], st["qkv"][:, H:H + KV], st["qkv"][:, H + KV:]
    cached = bool(c["cap"])
    if own:
        vrs = _vrs()
        _ctx.rope(q, k, st["freq"], rot_dim=rot, layout=vrs.ROPE_HALF if c["layout"] == "half" else vrs.ROPE_PAIRS,
                  seqs=st["seqs"], positions=st.get("positions"), axis_pairs=[hi - lo for lo, hi in _axes(c)],
                  q_out=st["q_out"], k_out=st["k_out"], v=v if cached else None, v_out=st["v_out"] if cached else None)
        return {"q": st["q_out"], "k": st["k_out"], **({"v": st["v_out"]} if cached else {})}
    n = st["rows"]
    seq, at = _rows(st)
    place = st["k_len"][seq].long() - (st["q_start"][seq + 1] - st["q_start"][seq]).long() + at
    if c["axes"] > 1:
        axis = torch.searchsorted(torch.tensor([hi for _, hi in _axes(c)], device=DEV),
                                  torch.arange(rot // 2, device=DEV), right=True)
        pos = st["positions"][:, :n].t().double()[:, axis]
    else:
        pos = place.double()[:, None]
    turn = pos * st["freq"]
    angle = (turn - torch.round(turn)) * (2 * math.pi)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x):
        x = x[:n].float()
        h = rot // 2
        a, b = (x[..., :h], x[..., h:rot]) if c["layout"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
        y0, y1 = a * cos - b * sin, a * sin + b * cos
        turned = torch.cat([y0, y1], -1) if c["layout"] == "half" else torch.stack([y0, y1], -1).flatten(-2)
        return torch.cat([turned, x[..., rot:]], -1).to(st["qkv"].dtype)

    to = st["k_start"][seq].long() + place
    st["q_out"][:n] = rotate(q)
    st["k_out"].index_copy_(0, to, rotate(k))
    if cached:
        st["v_out"].index_copy_(0, to, v[:n])
    return {"q": st["q_out"], "k": st["k_out"], **({"v": st["v_out"]} if cached else {})}


def _run_attention(st):
    c = st["case"]
    if own:
        _vrs()
        return _ctx.attention(st["q"], st["k"], st["v"], st["seqs"], causal=c["causal"], out=st["out"])
    H, KV, D, n = c["heads"], c["kv"], c["dim"], c["n"]
    G, MQ, MK = H // KV, st["max_q"], st["max_k"]
    # every sequence at the longest one's size, what lies past its own masked
    iq, ik = torch.arange(MQ, device=DEV), torch.arange(MK, device=DEV)
    q_len = (st["q_start"][1:] - st["q_start"][:-1]).long()
    k_len = st["k_len"].long()
    rows_q = (st["q_start"][:-1, None].long() + iq).clamp(max=st["q"].shape[0] - 1)
    rows_k = (st["k_start"][:, None].long() + ik).clamp(max=st["k"].shape[0] - 1)
    Q = st["q"][rows_q].float().view(n, MQ, KV, G, D).permute(0, 2, 3, 1, 4).reshape(n, KV, G * MQ, D)
    K = st["k"][rows_k].float().permute(0, 2, 3, 1).contiguous()
    V = st["v"][rows_k].float().permute(0, 2, 1, 3).contiguous()
    seen = ik[None, None, :] < k_len[:, None, None]
    if c["causal"]:
        seen = seen & (ik[None, None, :] <= (k_len - q_len)[:, None, None] + iq[None, :, None])
    s = torch.matmul(Q * D ** -0.5, K).view(n, KV, G, -1, MK)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, KV, G * MQ, MK), V).view(n, KV, G, MQ, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(n, MQ, H, D)
    seq, at = _rows(st)
    st["out"][:st["rows"]] = o[seq, at].to(st["out"].dtype)
    return st["out"]


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        x = st["x"].double()
        total = x if st["res"] is None else x + st["res"].double()
        y = total / torch.sqrt(torch.mean(total ** 2, dim=1, keepdim=True) + EPS) * st["weight"].double()
        r = {} if st["res"] is None else {"sum": total}
        if case["out"] == "same":
            return {"y": y, **r}
        if case["out"] == "step":
            return {"y": (y / st["step"]).clamp(-448, 448), **r}
        parts = y.split(case["cols"] if case["out"] == "row" else int(case["out"][5:]), dim=1)
        big = torch.stack([p.abs().max(dim=1).values for p in parts], dim=1)
        scale = torch.where(big == 0, torch.ones_like(big), big / 448)
        return {"y": torch.cat([p / scale[:, i:i + 1] for i, p in enumerate(parts)], dim=1), "scales": scale, **r}
    q_len, past = _lengths(case)
    H, KV, D = case["heads"], case["kv"], case["dim"]
    k_at = st["k_start"].tolist()
    if case["kind"] == "rope":
        qkv = st["qkv"].double()
        q_out, k_out, v_out = st["q_out"].double(), st["k_out"].double(), st["v_out"].double()
        half = case["rot"] // 2
        row = 0
        for i, (n, p) in enumerate(zip(q_len, past)):
            if case["axes"] > 1:
                pos = torch.cat([st["positions"][a, row:row + n, None].double().expand(n, hi - lo)
                                 for a, (lo, hi) in enumerate(_axes(case))], dim=1)
            else:
                pos = torch.arange(p, p + n, device=DEV, dtype=torch.float64)[:, None].expand(n, half)
            z = torch.polar(torch.ones(n, half, dtype=torch.float64, device=DEV), 2 * math.pi * torch.remainder(pos * st["freq"], 1.0))
            x = qkv[row:row + n, :H + KV].clone()
            pick = (slice(0, half), slice(half, 2 * half)) if case["layout"] == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
            w = torch.complex(x[..., pick[0]].contiguous(), x[..., pick[1]].contiguous()) * z[:, None]
            x[..., pick[0]], x[..., pick[1]] = w.real, w.imag
            q_out[row:row + n] = x[:, :H]
            to = slice(k_at[i] + p, k_at[i] + p + n)
            k_out[to], v_out[to] = x[:, H:], qkv[row:row + n, H + KV:]
            row += n
        return {"q": q_out, "k": k_out, **({"v": v_out} if case["cap"] else {})}
    out = st["out"].double()
    row = 0
    for i, (n, p) in enumerate(zip(q_len, past)):
        keys = slice(k_at[i], k_at[i] + p + n)
        hidden = torch.ones(n, p + n, dtype=torch.bool, device=DEV).triu(p + 1) if case["causal"] else None
        for h in range(H):
            k, v = st["k"][keys, h * KV // H].double(), st["v"][keys, h * KV // H].double()
            score = st["q"][row:row + n, h].double() @ k.t() / math.sqrt(D)
            if hidden is not None:
                score.masked_fill_(hidden, -math.inf)
            out[row:row + n, h] = torch.softmax(score, dim=1) @ v
        row += n
    return out

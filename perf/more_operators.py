"""Timing cases of the operators that generate from a cache on one MI355X: attention
of sequences that share a prefix, beam search's selection and the reordering of its
states, the attention that each key of a cache received, and eviction of the keys
that received least.

`listed()` holds the calls that stand for their uses, `draw()` further sizes of
the same ranges.  `run()` computes the operators in elementary torch operations
(32 bits; log-probabilities, whose order decides, in 64), or, where `own` is true,
by the calls that a program makes of this framework.  `exact()` restates each
definition in 64 bits.
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
TAIL = 3        # rows behind the last sequence: a program's buffers are longer than what one call fills
ROOM = 2        # rows of a sequence's place in the cache behind its last key

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


def _prefix(name, dtype, heads, kv, dim, groups, n, prefix, q, past, mix):
    """`groups` requests of n[0] .. n[1] sequences, each request with its own prefix."""
    return {"name": name, "kind": "prefix", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "groups": groups,
            "n_lo": n[0], "n_hi": n[1], "prefix_lo": prefix[0], "prefix_hi": prefix[1], "q_lo": q[0], "q_hi": q[1],
            "past_lo": past[0], "past_hi": past[1], "mix": mix}


def _select(name, dtype, batch, beams, vocab, k, done, mix):
    return {"name": name, "kind": "select", "dtype": dtype, "batch": batch, "beams": beams, "vocab": vocab, "k": k,
            "done": done, "mix": mix}


def _reorder(name, dtype, layers, batch, beams, kv, dim, rows, mix):
    return {"name": name, "kind": "reorder", "dtype": dtype, "layers": layers, "batch": batch, "beams": beams, "kv": kv,
            "dim": dim, "row_lo": rows[0], "row_hi": rows[1], "mix": mix}


def _weights(name, dtype, heads, kv, dim, n, q, past, decay, mix):
    return {"name": name, "kind": "weights", "dtype": dtype, "heads": heads, "kv": kv, "dim": dim, "n": n,
            "q_lo": q[0], "q_hi": q[1], "past_lo": past[0], "past_hi": past[1], "decay": decay, "mix": mix}


def _evict(name, dtype, kv, dim, n, keys, budget, first, recent, inplace, mix):
    return {"name": name, "kind": "evict", "dtype": dtype, "kv": kv, "dim": dim, "n": n, "k_lo": keys[0],
            "k_hi": keys[1], "budget": budget, "first": first, "recent": recent, "inplace": inplace, "mix": mix}


def listed():
    return [
        # the next token of five continuations of one prompt, float32, heads of 80: the smallest call, latency
        _prefix("prefix-samples-f32", "f32", 16, 4, 80, 1, (5, 5), (600, 600), (1, 1), (0, 30), 1),
        # the next token of four requests with 16 continuations each: bound by memory if the prefix is read once
        _prefix("prefix-samples-64", "bf16", 32, 8, 128, 4, (16, 16), (1500, 6000), (1, 1), (20, 700), 2),
        # 24 questions about one long document: bound by the matrix cores
        _prefix("prefix-questions", "bf16", 32, 8, 128, 1, (24, 24), (9000, 9000), (30, 200), (0, 0), 3),
        # the step of one request's four beams: latency
        _select("select-one", "bf16", 1, 4, 32000, 4, False, 4),
        # the step of 32 requests, some beams at their end, with twice as many candidates as beams
        _select("select-batch", "bf16", 32, 8, 128000, 16, True, 5),
        # float32 logits, a vocabulary that no vector divides
        _select("select-f32-odd", "f32", 5, 3, 50001, 6, True, 6),
        # keys and values of one request's beams behind their prompt, all layers: the smallest reordering
        _reorder("reorder-one", "bf16", 24, 1, 4, 2, 128, (7, 40), 7),
        # those of 16 requests
        _reorder("reorder-batch", "bf16", 16, 16, 8, 8, 128, (60, 300), 8),
        # what the tokens of 64 requests attended to: bound by memory
        _weights("weights-tokens-64", "bf16", 32, 8, 128, 64, (1, 1), (500, 8000), 1.0, 9),
        # what a prompt's queries attended to
        _weights("weights-prompt", "bf16", 32, 8, 128, 1, (4096, 4096), (0, 0), 1.0, 10),
        # one float32 cache cut to its budget: latency
        _evict("evict-one-f32", "f32", 4, 72, 1, (700, 700), 513, 4, 32, False, 11),
        # the caches of 16 requests cut to 2048 keys where they lie
        _evict("evict-batch", "bf16", 8, 128, 16, (2500, 8000), 2048, 4, 256, True, 12),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) if hi > lo else lo


def draw(rng):
    mix = rng.randrange(1 << 20)
    dtype = "bf16" if rng.random() < 0.7 else "f32"
    dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8] if dtype == "bf16" else [1, 2, 4])
    kind = rng.choice(["prefix", "prefix", "select", "select", "reorder", "weights", "evict"])
    if kind == "prefix":
        groups = _log(rng, 1, 12)
        n = _log(rng, 1, max(1, 96 // groups))
        if rng.random() < 0.6:      # single tokens, or a few
            prefix, past, q = _log(rng, 16, 9000), _log(rng, 1, 900), rng.choice([1, 1, 1, 2, 4])
            prefix = min(prefix, 400_000_000 // (groups * n * kv * dim))    # what the plain form holds
        else:
            q, past = _log(rng, 8, 300), rng.choice([0, 0, 100])
            prefix = _log(rng, 16, 9000)
            cost = groups * n * heads * q
            prefix = max(8, min(prefix, 24 * 200 * 32 * 9000 // 2 // cost, 400_000_000 // (groups * n * kv * dim)))
            q = min(q, max(8, 24 * 200 * 32 * 9000 // 2 // (groups * n * heads * prefix)))
        c = _prefix("", dtype, heads, kv, dim, groups, (max(1, n // rng.choice([1, 2])), n),
                    (max(1, prefix // rng.choice([1, 1, 4])), prefix), (max(1, q // rng.choice([1, 1, 4])), q),
                    (past // rng.choice([1, 2, 9]), past), mix)
    elif kind == "select":
        vocab, beams = _log(rng, 200, 260000), _log(rng, 1, 32)
        batch = max(1, min(_log(rng, 1, 64), 32 * 8 * 128000 // (vocab * beams * (2 if dtype == "f32" else 1))))
        k = min(64, max(1, beams * rng.choice([1, 1, 2])))
        c = _select("", dtype, batch, beams, vocab, k, rng.random() < 0.5, mix)
    elif kind == "reorder":
        layers, batch, beams = _log(rng, 1, 32), _log(rng, 1, 32), _log(rng, 2, 16)
        rows = max(1, min(_log(rng, 1, 600), 16 * 128 * 300 * 1024 // (layers * batch * beams * kv * dim * (2 if dtype == "f32" else 1))))
        c = _reorder("", dtype, layers, batch, beams, kv, dim, (max(1, rows // rng.choice([1, 2, 6])), rows), mix)
    elif kind == "weights":
        if rng.random() < 0.6:
            n, q = _log(rng, 1, 96), rng.choice([1, 1, 1, 3, 8])
            past = min(_log(rng, 1, 8000), 64 * 4200 * 8 * 128 * 2 // (n * kv * dim * ES[dtype]))
        else:
            n, past = _log(rng, 1, 24), rng.choice([0, 0, 500])
            q = min(4096 if dtype == "bf16" else 2000, int(math.sqrt(32 * 4096 * 4096 / 2 / (n * heads))))
            q = _log(rng, 16, max(17, q))
            past = min(past, 32 * 4096 * 4096 // 4 // (n * heads * q))
        c = _weights("", dtype, heads, kv, dim, n, (max(1, q // rng.choice([1, 2, 9])), q),
                     (past // rng.choice([1, 2, 5]), past), rng.choice([1.0, 1.0, 0.9375]), mix)
    else:
        n, keys = _log(rng, 1, 48), _log(rng, 20, 16000)
        keys = max(8, min(keys, 16 * 8000 * 8 * 128 * 2 // (n * kv * dim * ES[dtype])))
        budget = max(4, int(keys * rng.choice([0.2, 0.5, 0.9])))
        c = _evict("", dtype, kv, dim, n, (max(1, keys // rng.choice([1, 2, 4])), keys), budget,
                   rng.choice([0, 1, 4]), rng.choice([0, budget // 8, max(0, budget - 4)]), rng.random() < 0.5, mix)
    del c["name"]
    return c


# ---- lengths, as a program's scheduler knows them ------------------------------


def _lengths(case):
    """Group, queries and earlier keys of each sequence; each group's prefix."""
    r = random.Random(case["mix"])
    if case["kind"] == "prefix":
        sizes = [r.randint(case["n_lo"], case["n_hi"]) for _ in range(case["groups"])]
        prefix = [r.randint(case["prefix_lo"], case["prefix_hi"]) for _ in sizes]
    else:
        sizes, prefix = [1] * case["n"], []
    group = [i for i, s in enumerate(sizes) for _ in range(s)]
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in group]
    past = [r.randint(case["past_lo"], case["past_hi"]) for _ in group]
    return group, q, past, prefix


def _rows_of(case):
    """Rows of each slot that are in use (reorder: the same of a request's beams), or keys (evict)."""
    r = random.Random(case["mix"])
    if case["kind"] == "reorder":
        return [r.randint(case["row_lo"], case["row_hi"]) for _ in range(case["batch"])]
    return [r.randint(case["k_lo"], case["k_hi"]) for _ in range(case["n"])]


def _parents(case, r):
    """What a step's selection gives: the best beams go on, some of them twice."""
    return [sorted(min(int(r.expovariate(1.6) * case["beams"] / 2), case["beams"] - 1) for _ in range(case["beams"]))
            for _ in range(case["batch"])]


def work(case):
    es, kind = ES.get(case["dtype"], 4), case["kind"]
    if kind == "select":
        rows = case["batch"] * case["beams"]
        read = rows * case["vocab"] * (0.75 if case["done"] else 1)
        return {"bytes": read * es + 5 * rows + 12 * case["batch"] * case["k"], "flops": 4 * read}
    if kind == "reorder":
        lens, row = _rows_of(case), case["layers"] * 2 * case["kv"] * case["dim"] * es
        move = 0
        for n, p in zip(lens, _parents(case, random.Random(case["mix"] + 1))):
            moved = [i for i in range(case["beams"]) if p[i] != i]
            move += n * (len(moved) + len({p[i] for i in moved}))      # each parent read once
        return {"bytes": move * row + 4 * case["batch"] * case["beams"], "flops": 0}
    if kind == "evict":
        lens = _rows_of(case)
        left = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": case["kv"] * (4 * sum(lens) + left * (2 * 2 * case["dim"] * es + 4 + 4)), "flops": 0}
    group, q, past, prefix = _lengths(case)
    causal = sum(a * (p + a) - a * (a - 1) // 2 for a, p in zip(q, past))
    own_keys = sum(q) + sum(past)
    if kind == "prefix":
        pairs = causal + sum(a * prefix[g] for a, g in zip(q, group))
        keys = own_keys + sum(prefix)
        return {"bytes": es * case["dim"] * (2 * sum(q) * case["heads"] + 2 * keys * case["kv"]),
                "flops": 4 * case["dim"] * case["heads"] * pairs}
    return {"bytes": es * case["dim"] * (sum(q) * case["heads"] + own_keys * case["kv"]) + 8 * own_keys * case["kv"],
            "flops": 2 * case["dim"] * case["heads"] * causal}


# ---- inputs ---------------------------------------------------------------------


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, kind = TDT[case["dtype"]], case["kind"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dt)

    st = {"case": case}
    if kind == "select":
        batch, beams, vocab = case["batch"], case["beams"], case["vocab"]
        # what a language model's last product gives: a bulk, and some dozens of tokens that fit
        logits = torch.randn(batch, beams, vocab, generator=g, device=DEV) * 2
        fit = torch.randint(0, vocab, (batch, beams, min(48, vocab)), generator=g, device=DEV)
        logits.scatter_add_(2, fit, torch.rand(fit.shape, generator=g, device=DEV) * 12)
        logits[..., : vocab // 97] = -math.inf         # tokens that a grammar forbids
        st["logits"] = logits.to(dt)
        st["scores"] = -torch.rand(batch, beams, generator=g, device=DEV).mul(9).cumsum(1)
        done = torch.rand(batch, beams, generator=g, device=DEV) < 0.25
        st["done"] = done.to(torch.uint8) if case["done"] else None
        st["eos"] = vocab - 1
        return st
    if kind == "reorder":
        lens = _rows_of(case)
        room = case["row_hi"] + ROOM
        st["state"] = normal(case["layers"], case["batch"] * case["beams"], room, 2 * case["kv"] * case["dim"])
        r = random.Random(case["mix"] + 1)
        st["parents"] = _i32(_parents(case, r))
        st["len"] = _i32([n for n in lens for _ in range(case["beams"])])
        return st
    if kind == "evict":
        lens, kv, dim, n = _rows_of(case), case["kv"], case["dim"], case["n"]
        cap = max(case["k_hi"], case["budget"]) + ROOM
        st["cap"], st["max_k"] = cap, case["k_hi"]
        st["k_start"], st["k_len"] = _i32([i * cap for i in range(n)]), _i32(lens)
        st["k"], st["v"] = normal(n * cap, kv, dim), normal(n * cap, kv, dim)
        # weights that add up over many steps: a few keys have most; those never attended to have none
        acc = torch.exp(2 * torch.randn(kv, n * cap, generator=g, device=DEV))
        st["acc"] = torch.where(torch.rand(kv, n * cap, generator=g, device=DEV) < 0.1, torch.zeros_like(acc), acc)
        fresh = not case["inplace"]
        st["k_out"], st["v_out"] = (torch.zeros_like(st["k"]), torch.zeros_like(st["v"])) if fresh else (st["k"], st["v"])
        st["acc_out"] = torch.zeros_like(st["acc"]) if fresh else st["acc"]
        st["len_out"] = torch.zeros_like(st["k_len"])
        st["kept"] = torch.zeros(n, kv, case["budget"], dtype=torch.int32, device=DEV)
        return st
    group, q, past, prefix = _lengths(case)
    k_len = [a + b for a, b in zip(q, past)]
    H, KV, D, n = case["heads"], case["kv"], case["dim"], len(q)
    starts = [sum(q[:i]) for i in range(n + 1)]
    cap = case["q_hi"] + case["past_hi"] + ROOM
    base = sum(prefix) + len(prefix)      # the prefixes lie before the sequences' own places
    st["q_start"], st["k_len"] = _i32(starts), _i32(k_len)
    st["k_start"] = _i32([base + i * cap for i in range(n)])
    st["rows"], st["max_q"], st["max_k"] = sum(q), max(q), max(k_len)
    k_rows = base + n * cap
    st["q"] = normal(sum(q) + TAIL, H, D, scale=2.0)      # scores with some weight on single keys
    st["k"] = normal(k_rows, KV, D)
    if kind == "weights":
        st["acc"] = torch.rand(KV, k_rows, generator=g, device=DEV)
    else:
        st["v"] = normal(k_rows, KV, D)
        st["out"] = torch.full((sum(q) + TAIL, H, D), 1 / 64, dtype=dt, device=DEV)
        st["p_start"] = _i32([sum(prefix[:i]) + i for i in range(len(prefix))])
        st["p_len"] = _i32(prefix)
        st["first"] = _i32([sum(1 for x in group if x < i) for i in range(len(prefix) + 1)])
        st["group"] = _i32(group).long()
        st["max_prefix"] = max(prefix)
        rows = [sum(a for a, x in zip(q, group) if x == i) for i in range(len(prefix))]
        st["max_rows"] = max(rows)
    if own:      # the plan of the batch, which a program makes once and uses in every layer
        vrs = _vrs()
        st["seqs"] = vrs.seqs(st["q_start"], st["k_start"], st["k_len"], max_q=st["max_q"], max_k=st["max_k"])
        if kind == "prefix":
            st["prefixes"] = vrs.prefixes(st["first"], st["p_start"], st["p_len"], max_rows=st["max_rows"],
                                          max_k=st["max_prefix"])
    return st


# ---- the operators ----------------------------------------------------------------


def run(st):
    return {"prefix": _run_prefix, "select": _run_select, "reorder": _run_reorder, "weights": _run_weights,
            "evict": _run_evict}[st["case"]["kind"]](st)


def _softmax_parts(st, rows_k, seen):
    """Queries of every sequence at the longest one's size, and exp(score - maximum) over the keys in rows
    `rows_k` [n, keys] that `seen` [n, MQ, keys] lets them see."""
    c = st["case"]
    H, KV, D, MQ = c["heads"], c["kv"], c["dim"], st["max_q"]
    n, MK = rows_k.shape
    G = H // KV
    iq = torch.arange(MQ, device=DEV)
    rows_q = (st["q_start"][:-1, None].long() + iq).clamp(max=st["q"].shape[0] - 1)
    Q = st["q"][rows_q].float().view(n, MQ, KV, G, D).permute(0, 2, 3, 1, 4).reshape(n, KV, G * MQ, D)
    K = st["k"][rows_k].float().permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(Q * D ** -0.5, K).view(n, KV, G, MQ, MK)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    return p, p.sum(-1, keepdim=True)


def _own_keys(st):
    """Rows of each sequence's own keys at the longest one's size, and which of them its queries see."""
    iq, ik = torch.arange(st["max_q"], device=DEV), torch.arange(st["max_k"], device=DEV)
    q_len = (st["q_start"][1:] - st["q_start"][:-1]).long()
    k_len = st["k_len"].long()
    rows = (st["k_start"][:, None].long() + ik).clamp(max=st["k"].shape[0] - 1)
    has = ik[None] < k_len[:, None]
    own_place = (k_len - q_len)[:, None, None] + iq[None, :, None]
    return rows, has, has[:, None] & (ik[None, None] <= own_place), iq[None] < q_len[:, None]


def _run_prefix(st):
    if own:
        _vrs()
        return _ctx.prefix_attention(st["q"], st["k"], st["v"], st["seqs"], st["prefixes"], out=st["out"])
    c = st["case"]
    H, KV, D, MQ = c["heads"], c["kv"], c["dim"], st["max_q"]
    n = st["k_len"].numel()
    rows, _, seen, is_q = _own_keys(st)
    ip = torch.arange(st["max_prefix"], device=DEV)
    rows_p = (st["p_start"].long()[:, None] + ip).clamp(max=st["k"].shape[0] - 1)[st["group"]]
    seen_p = (ip[None] < st["p_len"][:, None])[st["group"]]
    rows_k = torch.cat([rows_p, rows], 1)
    p, total = _softmax_parts(st, rows_k, torch.cat([seen_p[:, None].expand(n, MQ, -1), seen], 2))
    V = st["v"][rows_k].float().permute(0, 2, 1, 3).contiguous()
    o = torch.matmul(p.view(n, KV, -1, rows_k.shape[1]), V).view(n, KV, H // KV, MQ, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(n, MQ, H, D)
    seq, at = _places(st)
    st["out"][:st["rows"]] = o[seq, at].to(st["out"].dtype)
    return st["out"]


def _places(st):
    """Sequence and place in it of each query row."""
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(st["q_start"][1:].long(), row, right=True)
    return seq, row - st["q_start"][seq].long()


def _run_select(st):
    c = st["case"]
    if own:
        _vrs()
        s, parents, tokens = _ctx.beam_select(st["logits"], st["scores"], c["k"], done=st["done"], eos=st["eos"])
        return {"scores": s, "parents": parents, "tokens": tokens}
    x = st["logits"].double()
    m = x.amax(-1, keepdim=True)
    lse = m + (x - m).exp().sum(-1, keepdim=True).log()
    cand = st["scores"].double()[..., None] + (x - lse)
    if st["done"] is not None:      # a beam at its end goes on with the end token alone, at no cost
        only = torch.full_like(cand, -math.inf)
        only[..., st["eos"]] = st["scores"].double()
        cand = torch.where(st["done"].bool()[..., None], only, cand)
    cand = torch.where(cand.isnan(), torch.full_like(cand, -math.inf), cand).flatten(1)
    best, at = torch.sort(cand, dim=1, descending=True, stable=True)
    best, at = best[:, :c["k"]], at[:, :c["k"]]
    return {"scores": best.float(), "parents": (at // c["vocab"]).int(), "tokens": (at % c["vocab"]).int()}


def _run_reorder(st):
    c, state = st["case"], st["state"]
    if own:
        _vrs()
        _ctx.beam_reorder(state, st["parents"], lens=st["len"])
        return state
    x = state.view(c["layers"], c["batch"], c["beams"], state.shape[2], -1)
    b = torch.arange(c["batch"], device=DEV)[:, None]
    used = torch.arange(state.shape[2], device=DEV) < st["len"].view(c["batch"], c["beams"])[b, st["parents"].long()][..., None]
    x.copy_(torch.where(used[None, ..., None], x[:, b, st["parents"].long()], x))
    return state


def _run_weights(st):
    c, acc = st["case"], st["acc"]
    if own:
        _vrs()
        _ctx.attention_weights(st["q"], st["k"], st["seqs"], acc, decay=c["decay"])
        return acc
    rows, has, seen, is_q = _own_keys(st)
    p, total = _softmax_parts(st, rows, seen)
    p = p.mul_(torch.where(total > 0, 1 / total, torch.zeros_like(total))).mul_(is_q[:, None, None, :, None])
    w = p.sum((2, 3)) * has[:, None]                # [n, KV, keys]
    flat = rows.flatten()
    add = torch.zeros_like(acc).index_add_(1, flat, w.permute(1, 0, 2).reshape(c["kv"], -1))
    covered = torch.zeros(acc.shape[1], device=DEV).index_add_(0, flat, has.flatten().float()) > 0
    acc.copy_(torch.where(covered, acc * c["decay"], acc) + add)
    return acc


def _run_evict(st):
    c, budget = st["case"], st["case"]["budget"]
    names = ("k_out", "v_out", "acc_out", "len_out", "kept")
    if own:
        _vrs()
        _ctx.cache_evict(st["k"], st["v"], st["acc"], st["k_start"], st["k_len"], budget, first=c["first"],
                         recent=c["recent"], max_k=st["max_k"], k_out=st["k_out"], v_out=st["v_out"],
                         acc_out=st["acc_out"], len_out=st["len_out"], kept=st["kept"])
        return {x: st[x] for x in names}
    n, kv = c["n"], c["kv"]
    ik = torch.arange(max(st["max_k"], budget), device=DEV)
    k_len = st["k_len"].long()[:, None]
    rows = st["k_start"].long()[:, None] + ik
    inside = ik < k_len
    forced = ((ik < c["first"]) | (ik >= k_len - c["recent"])) & inside
    a = st["acc"][:, rows].permute(1, 0, 2)          # [n, kv, keys]
    a = torch.where(forced[:, None], math.inf, torch.where(inside[:, None], a, -math.inf))
    at = torch.sort(a, dim=2, descending=True, stable=True)[1][..., :budget]
    new_len = k_len.clamp(max=budget)
    j = torch.arange(budget, device=DEV)
    at = torch.sort(torch.where(j < new_len[:, None], at, ik.numel()), dim=2)[0]
    live = (j < new_len)[:, None].expand(n, kv, budget)
    src = (st["k_start"].long()[:, None, None] + at.clamp(max=ik.numel() - 1)).clamp(max=st["k"].shape[0] - 1)
    dst = (st["k_start"].long()[:, None] + j)[:, None].expand(n, kv, budget)
    h = torch.arange(kv, device=DEV)[None, :, None]
    for x, y in (("k", "k_out"), ("v", "v_out")):
        st[y][dst, h] = torch.where(live[..., None], st[x][src, h], st[y][dst, h])
    st["acc_out"][h, dst] = torch.where(live, st["acc"][h, src], st["acc_out"][h, dst])
    st["kept"].copy_(torch.where(live, at, -1))
    st["len_out"].copy_(new_len[:, 0])
    return {x: st[x] for x in names}


# ---- the definitions in 64 bits -----------------------------------------------------


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "select":
        found = []
        for b in range(case["batch"]):
            lists = []
            for i in range(case["beams"]):
                s = st["scores"][b, i].double()
                if case["done"] and st["done"][b, i]:
                    c = torch.full((case["vocab"],), -math.inf, dtype=torch.float64, device=DEV)
                    c[st["eos"]] = s
                else:
                    c = s + torch.log_softmax(st["logits"][b, i].double(), 0)
                lists.append(c)
            found.append(torch.cat(lists).sort(descending=True).values[:case["k"]])
        return {"scores": torch.stack(found), "parents": None, "tokens": None}
    if kind == "reorder":
        state, beams = st["state"].double(), case["beams"]
        old = state.clone()
        for b, (n, p) in enumerate(zip(_rows_of(case), st["parents"].tolist())):
            for i, x in enumerate(p):
                state[:, b * beams + i, :n] = old[:, b * beams + x, :n]
        return state
    if kind == "evict":
        out = {"k_out": st["k_out"].double(), "v_out": st["v_out"].double(), "acc_out": st["acc_out"].double()}
        for i, n in enumerate(_rows_of(case)):
            left = min(n, case["budget"])
            a, to = int(st["k_start"][i]), slice(int(st["k_start"][i]), int(st["k_start"][i]) + left)
            for h in range(case["kv"]):
                acc = st["acc"][h, a:a + n].double().cpu().tolist()
                must = [j for j in range(n) if j < case["first"] or j >= n - case["recent"]]
                rest = sorted(set(range(n)) - set(must), key=lambda j: (-acc[j], j))
                keep = torch.tensor(sorted((must + rest[:max(0, left - len(must))])[:left]), dtype=torch.long, device=DEV)
                out["k_out"][to, h], out["v_out"][to, h] = st["k"][a + keep, h].double(), st["v"][a + keep, h].double()
                out["acc_out"][h, to] = st["acc"][h, a + keep].double()
        return {**out, "len_out": None, "kept": None}
    group, q_len, past, prefix = _lengths(case)
    H, KV, D = case["heads"], case["kv"], case["dim"]
    if H * sum(a * (a + b) for a, b in zip(q_len, past)) * D > 3e13:
        return None
    k_at = st["k_start"].tolist()
    p_at = st["p_start"].tolist() if kind == "prefix" else []
    res = st["out"].double() if kind == "prefix" else st["acc"].double()
    row = 0
    for i, (n, p) in enumerate(zip(q_len, past)):
        lead = prefix[group[i]] if kind == "prefix" else 0
        keys = torch.arange(k_at[i], k_at[i] + p + n, device=DEV)
        if kind == "prefix":
            keys = torch.cat([torch.arange(p_at[group[i]], p_at[group[i]] + lead, device=DEV), keys])
        else:
            res[:, keys] *= case["decay"]
        hidden = torch.ones(n, lead + p + n, dtype=torch.bool, device=DEV).triu(lead + p + 1)
        for h in range(KV):
            mine = slice(h * H // KV, (h + 1) * H // KV)
            k = st["k"][keys, h].double()
            score = st["q"][row:row + n, mine].double().transpose(0, 1) @ k.t() / math.sqrt(D)
            w = torch.softmax(score.masked_fill_(hidden, -math.inf), dim=2)
            if kind == "prefix":
                res[row:row + n, mine] = (w @ st["v"][keys, h].double()).transpose(0, 1)
            else:
                res[h, keys] += w.sum((0, 1))
        row += n
    return res

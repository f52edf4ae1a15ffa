"""Operators that generate from a cache (attention over shared prefixes, beam
search's step, attention that keys receive, eviction) against their definitions in
64 bits, at the sizes, strides and masks where they can go wrong, and a run of them
together.

Tolerances count roundings: a type rounds by at most U[type] of the value
(bfloat16 2^-8, float32 2^-24), a float32 sum of n terms by n 2^-24 of the sum of
their magnitudes."""
import math

import numpy as np
import pytest

from gpu_util import ctx, vrs
from test_gpu_transformer import F, U, i32, inside, randn, tdt

pytestmark = pytest.mark.gpu


def replayed(call, outs, reset, times=3):
    """What `outs` hold after each of several replays of a captured call, with eager work between."""
    import torch
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    got = []
    for _ in range(times):
        reset()
        torch.cuda.synchronize()
        g.replay()
        got.append([o.clone() for o in outs])
        torch.randn(1000, device="cuda").sum().item()
    return got


# ---- attention over shared prefixes --------------------------------------------------

# queries and earlier own keys of each sequence; sequences of each group; prefixes
GROUPS = {
    "tokens": ([1] * 7, [5, 0, 33, 64, 1, 200, 7], [0, 3, 7], [300, 40]),
    "one": ([1], [0], [0, 1], [1]),
    "edges": ([1, 2, 0, 3, 1, 1], [0, 4, 9, 31, 32, 2], [1, 1, 4, 5], [77, 33, 0]),        # sequences of no group, empty ones
    "prompts": ([40, 130, 1, 65], [0, 0, 3, 10], [0, 2, 4], [129, 500]),
    "short": ([5, 9, 2], [-3, -20, 0], [0, 3], [10]),                                      # fewer own keys than queries
    "many": ([1] * 140, [i % 9 for i in range(140)], [2 * i for i in range(71)], [3 * i for i in range(70)]),
    "group": ([1] * 40, [3] * 40, [0, 40], [1000]),
}


def build(case, lead=2, tail=3, hint=True):
    q_len, past, first, prefix = GROUPS[case] if isinstance(case, str) else case
    starts = [lead + sum(q_len[:i]) for i in range(len(q_len) + 1)]
    k_len = [max(0, a + b) for a, b in zip(q_len, past)]
    p_at = [int(x) for x in np.cumsum([1] + [p + 2 for p in prefix])]
    k_at = [int(x) for x in np.cumsum([p_at[-1]] + [n + 3 for n in k_len])]
    rows = [starts[b] - starts[a] for a, b in zip(first[:-1], first[1:])]
    h = dict(max_q=max(q_len), max_k=max(k_len)) if hint else {}
    hp = dict(max_rows=max(rows), max_k=max(prefix)) if hint else {}
    s = vrs.seqs(i32(starts), i32(k_at[:-1]), i32(k_len), **h)
    p = vrs.prefixes(i32(first), i32(p_at[:-1]), i32(prefix), **hp)
    group = [next((g for g in range(len(prefix)) if first[g] <= i < first[g + 1]), -1) for i in range(len(q_len))]
    return dict(q_len=q_len, starts=starts, rows=starts[-1] + tail, k_len=k_len, k_at=k_at, p_at=p_at, prefix=prefix,
                group=group, seqs=s, prefixes=p, k_rows=k_at[-1] + 2)


def prefix_ref(b, q, k, v, causal, scale, out, dtype):
    """Result and tolerance in 64 bits; `out` holds what rows of no sequence have."""
    import torch
    ref, tol = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64, device=out.device)
    H, G, D = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
    dev = q.device
    for i, n_own in enumerate(b["k_len"]):
        r0, r1, g = b["starts"][i], b["starts"][i + 1], b["group"][i]
        if r0 == r1:
            continue
        n_pre = b["prefix"][g] if g >= 0 else 0
        at = torch.cat([torch.arange(b["p_at"][g], b["p_at"][g] + n_pre, device=dev),
                        torch.arange(b["k_at"][i], b["k_at"][i] + n_own, device=dev)]).long()
        n = at.numel()
        Q = q[r0:r1].double().transpose(0, 1)
        K, V = (t[at].double().repeat_interleave(G, 1).transpose(0, 1) for t in (k, v))
        own = torch.arange(n, device=dev)[None] - n_pre
        seen = own <= (n_own - (r1 - r0) + torch.arange(r1 - r0, device=dev))[:, None] if causal else own < n_own
        seen = (seen | (own < 0)).expand(r1 - r0, n)
        s = (Q @ K.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        m = s.amax(2, keepdim=True) if n else s.new_full((H, r1 - r0, 1), -math.inf)
        p = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), 0.0)
        total = p.sum(2, keepdim=True)
        Vs = torch.where(V.isfinite(), V, torch.zeros_like(V))
        w = p / torch.where(total == 0, torch.ones_like(total), total)
        o = w @ Vs
        for value in (math.inf, -math.inf, math.nan):      # counted apart, since 0 * inf is no 0
            hit = V.isnan() if value != value else V == value
            if hit.any():
                o = torch.where((seen.double()[None] @ hit.double()) > 0, o + value, o)
        # as vrs_attention's: probabilities rounded by u, scores off by e, float32 sums; and the join of up to 80
        # parts, whose factors are off by 4 units each and whose sums by one a part
        u = 0.0 if dtype == "f32" else U["bf16"]
        if n:
            big = (Q.abs() @ K.abs().transpose(1, 2) * scale).masked_fill(~seen, 0).amax(2, keepdim=True)
            e = (D + 8) * F * big + 8 * F
            of = o.nan_to_num(0, 0, 0)
            spread = torch.stack([(w[h][:, :, None] * (Vs[h][None] - of[h][:, None]).abs()).sum(1) for h in range(H)])
            t = spread * (u + 2 * e) * 1.02 + (w @ Vs.abs()) * (2 * n + 70 + 84) * F + of.abs() * U[dtype] * 1.01
        else:
            t = torch.zeros_like(o)
        ref[r0:r1], tol[r0:r1] = o.transpose(0, 1), t.transpose(0, 1)
    return ref, tol


def prefix_inputs(b, dtype, heads, kv, dim, seed=0):
    import torch
    q, k, v = (randn(b["rows"], heads, dim, dtype=dtype, seed=seed, scale=2), randn(b["k_rows"], kv, dim, dtype=dtype, seed=seed + 1),
               randn(b["k_rows"], kv, dim, dtype=dtype, seed=seed + 2))
    return q, k, v, torch.full((b["rows"], heads, dim), 5.0, dtype=tdt(dtype), device="cuda")


def check_prefix(case, dtype="bf16", heads=4, kv=2, dim=64, causal=True, scale=0.0, hint=True, seed=0, edit=None):
    import torch
    b = build(case, hint=hint)
    q, k, v, out = prefix_inputs(b, dtype, heads, kv, dim, seed)
    if edit:
        edit(b, q, k, v)
    ref, tol = prefix_ref(b, q, k, v, causal, scale or dim ** -0.5, out, dtype)
    got = ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], causal=causal, scale=scale, out=out)
    torch.cuda.synchronize()
    assert got is out
    inside(got, ref, tol)
    return b, q, k, v, out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", list(GROUPS))
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (3, 3, 8), (8, 1, 128), (5, 1, 72)])
def test_prefix_attention(dtype, causal, case, heads, kv, dim):
    check_prefix(case, dtype, heads, kv, dim, causal)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 127, 129, 257, 5000])
def test_prefix_attention_lengths(dtype, n):
    """Prefixes around the sizes of the tiles, read by few rows, by many, and by prompts."""
    check_prefix(([1, 1, 1], [2, 40, 0], [0, 3], [n]), dtype, 8, 2, 64, seed=n)
    check_prefix(([1] * 24, [n % 50] * 24, [0, 24], [n]), dtype, 8, 2, 128, seed=n)
    check_prefix(([70, 3, 31], [0, 5, 0], [0, 3], [n]), dtype, 4, 2, 64, seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_attention_large(dtype):
    """Many key tiles and parts, groups of unequal lengths."""
    check_prefix(([1] * 20, [300 + 37 * i for i in range(20)], [0, 2, 20], [9000, 700]), dtype, 8, 2, 128)
    check_prefix(([1] * 100, [17] * 100, [0, 100], [3000]), dtype, 8, 2, 64)
    check_prefix(([300, 1, 200], [0, 900, 50], [0, 1, 3], [2500, 1100]), dtype, 4, 2, 128)


def test_prefix_attention_equals_attention_without_prefixes():
    """No groups: vrs_attention's own bits; groups of no keys: the same numbers to the join's rounding."""
    import torch
    b = build(([3, 1, 40], [60, 7, 0], [0, 3], [4]))
    q, k, v, out = prefix_inputs(b, "bf16", 4, 2, 64)
    want = ctx().attention(q, k, v, b["seqs"], out=out.clone())
    none = vrs.prefixes(i32([0]), i32([]), i32([]))
    assert torch.equal(ctx().prefix_attention(q, k, v, b["seqs"], none, out=out.clone()), want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", ["tokens", "prompts", "group"])
def test_prefix_attention_values_that_are_not_finite(dtype, case):
    """Infinities and NaN behind the prefix and the own keys, and in keys that a query does not see, touch nothing;
    values that are seen reach those that see them."""
    def edit(b, q, k, v):
        for g, n in enumerate(b["prefix"]):
            k[b["p_at"][g] + n], v[b["p_at"][g] + n] = math.nan, math.inf
        for i, n in enumerate(b["k_len"]):
            k[b["k_at"][i] + n], v[b["k_at"][i] + n] = math.inf, math.nan
        v[b["k_at"][0] + b["k_len"][0] - 1, 0, 3] = math.inf       # the last key: its last query alone
        v[b["p_at"][0], 1, 5] = -math.inf                          # all of the group
    check_prefix(case, dtype, edit=edit)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_keys_at_their_queries_rows(dtype):
    """Sequences without k_start and k_len: own keys lie at the queries' rows, prefixes behind them."""
    import torch
    for q_len, first, prefix in (([1, 1, 1], [0, 3], [50]), ([40, 130, 7], [0, 1, 3], [33, 200])):
        starts = [2 + sum(q_len[:i]) for i in range(len(q_len) + 1)]
        rows = starts[-1] + 3
        p_at = [rows + 1 + sum(prefix[:i]) for i in range(len(prefix))]
        b = dict(starts=starts, rows=rows, k_len=q_len, k_at=starts[:-1], p_at=p_at, prefix=prefix, k_rows=p_at[-1] + prefix[-1] + 2,
                 group=[next(g for g in range(len(prefix)) if first[g] <= i < first[g + 1]) for i in range(len(q_len))])
        seqs = vrs.seqs(i32(starts), max_q=max(q_len), max_k=max(q_len))
        q, k, v, out = prefix_inputs(b, dtype, 4, 2, 64)
        ref, tol = prefix_ref(b, q, k, v, True, 0.125, out, dtype)
        inside(ctx().prefix_attention(q, k, v, seqs, vrs.prefixes(i32(first), i32(p_at), i32(prefix)), out=out), ref, tol)
        acc = torch.rand(2, b["k_rows"], device="cuda")
        ref, tol = weights_ref(q, k, acc, starts, q_len, starts[:-1], True, 0.125, 0.5)
        inside(ctx().attention_weights(q, k, seqs, acc, decay=0.5), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_attention_scores_of_minus_infinity(dtype):
    """A query all of whose keys score -infinity is NaN, one that sees no key 0, and one run of such keys weighs nothing."""
    import torch
    b = build(([1, 1, 1], [4, 4, -1], [0, 1, 2, 3], [40, 40, 0]))
    q, k, v, out = prefix_inputs(b, dtype, 2, 1, 64)
    q[...] = 0
    q[..., 0] = 1
    k[b["p_at"][0]:b["p_at"][0] + 40, :, 0] = -math.inf
    k[b["p_at"][1]:b["p_at"][1] + 40, :, 0] = -math.inf
    k[b["k_at"][1]:b["k_at"][1] + 5, :, 0] = -math.inf
    k[..., 1:] = 0
    got = ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=out)
    own = ctx().attention(q, k, v, b["seqs"], out=out.clone())
    inside(got[2], own[2].double(), own[2].double().abs() * 2 * U[dtype] + 200 * F)
    assert got[3].isnan().all() and torch.all(got[4] == 0)


def test_prefix_attention_over_its_queries():
    """out may be q; few and many sequences, tokens and prompts."""
    import torch
    for case in ("tokens", "prompts", "many", "group", ([1] * 3, [700, 900, 40], [0, 3], [3000]), ([1] * 90, [9] * 90, [0, 45, 90], [400, 2000])):
        b = build(case)
        q, k, v, _ = prefix_inputs(b, "bf16", 32, 4, 128)
        want = ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=q.clone())
        ref, tol = prefix_ref(b, q, k, v, True, 128 ** -0.5, q, "bf16")
        inside(want, ref, tol)
        assert torch.equal(ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=q), want)


def test_prefix_attention_far_scores():
    """Prefix and own keys whose scores lie far from each other: the larger take all."""
    for dtype in ("bf16", "f32"):
        for to in ("p_at", "k_at"):
            def edit(b, q, k, v):
                q[..., 0] = 2.0 ** 17
                k[..., 0] = 0
                k[b[to][0]:b[to][0] + 5, :, 0] = 2.0 ** 17
            b = build(([1, 1, 1], [30, 30, 30], [0, 3], [200]))
            q, k, v, out = prefix_inputs(b, dtype, 4, 2, 64)
            q[..., 1:], k[..., 1:] = 0, 0
            edit(b, q, k, v)
            ref, _ = prefix_ref(b, q, k, v, True, 1.0, out, dtype)
            got = ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], scale=1.0, out=out)
            inside(got, ref, ref.abs() * U[dtype] * 2.02 + 300 * F * 6)


def test_prefix_attention_hints_choose_kernels_only():
    for case in ("tokens", "prompts", "group"):
        b = build(case)
        q, k, v, out = prefix_inputs(b, "bf16", 4, 2, 64)
        ref, tol = prefix_ref(b, q, k, v, True, 0.125, out, "bf16")
        for a in ((0, 0, 0, 0), (1, 1, 1, 1), (1, 0, 1 << 30, 1 << 30), (1 << 30, 1 << 30, 1, 5000), (64, 1, 40, 1)):
            b["seqs"].max_q, b["seqs"].max_k, b["prefixes"].max_rows, b["prefixes"].max_k = a
            inside(ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=out.clone()), ref, tol)


def test_prefix_attention_writes_no_row_outside():
    """Groups, starts and lengths that do not fit the buffers are cut off."""
    import torch
    for first, p_at, p_len in (([-4, 2, 900], [0, 5], [4, 4]), ([0, 2, 3], [-7, 1 << 30], [3, 3]), ([0, 3, 3], [35, 0], [1 << 30, -5])):
        q, k = randn(12, 2, 64, seed=1), randn(40, 1, 64, seed=2)
        big = torch.full((20, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
        s = vrs.seqs(i32([0, 4, 8, 500]), i32([20, 24, 28]), i32([4, 4, 4]))
        ctx().prefix_attention(q, k, k, s, vrs.prefixes(i32(first), i32(p_at), i32(p_len)), out=big[4:16])
        torch.cuda.synchronize()
        assert torch.all(big[:4] == 7) and torch.all(big[16:] == 7)
        assert not big[4:16].isnan().any()


def test_prefix_attention_strides_workspace_and_graph():
    """Views of one product, a workspace full of NaN, a side stream, replays that follow the lengths."""
    import torch
    b = build("tokens")
    qkv = randn(b["rows"], 4 + 2, 64, seed=1)
    kv = randn(b["k_rows"], 2, 2, 64, seed=2)
    q, k, v = qkv[:, :4], kv[:, 0], kv[:, 1]
    out = torch.full((b["rows"], 2, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")[:, 1]
    ref, tol = prefix_ref(b, q, k, v, True, 0.125, out, "bf16")
    d, _ = ctx()._attention_desc("x", q, k, v, True, 0.0, out, None)
    need = vrs.lib().vrs_prefix_attention_workspace_size(d, b["seqs"].address, b["prefixes"].address)
    ws = torch.full((need // 4,), math.nan, device="cuda").view(torch.uint8)
    call = lambda: ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=out, workspace=ws)   # noqa: E731
    call()
    inside(out, ref, tol)
    with pytest.raises(vrs.VrsError):
        ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], workspace=ws[:-16])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"])
    s.synchronize()
    assert torch.equal(other[2:-3], out[2:-3])
    want = out.clone()
    for (got,) in replayed(call, [out], lambda: out.fill_(5.0)):
        assert torch.equal(got, want)
    b["prefixes"].tensors[2].copy_(i32([290, 40]))         # the captured call would see these
    b["prefix"] = [290, 40]
    ref, tol = prefix_ref(b, q, k, v, True, 0.125, torch.full_like(out, 5.0), "bf16")
    for (got,) in replayed(call, [out], lambda: out.fill_(5.0)):
        inside(got, ref, tol)


# ---- beam search: the selection --------------------------------------------------------


def select_ref(logits, scores, k, done=None, eos=-1):
    """The k best in 64 bits on the CPU, equal ones by their place."""
    import torch
    x, s = logits.double().cpu(), scores.double().cpu()
    batch, beams, vocab = x.shape
    m = x.amax(2, keepdim=True)
    c = s[..., None] + (x - (m + (x - m).exp().sum(2, keepdim=True).log()))
    if done is not None:
        only = torch.full_like(c, -math.inf)
        only[..., eos] = s
        c = torch.where(done.bool().cpu()[..., None], only, c)
    fine = s.isfinite()[..., None] & ~c.isnan()
    c = torch.where(fine, c, torch.full_like(c, -math.inf)).flatten(1)
    best, at = torch.sort(c, dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    return best, (at // vocab).int(), (at % vocab).int()


def check_select(logits, scores, k, done=None, eos=-1, **kw):
    import torch
    ref = select_ref(logits, scores, k, done, eos)
    got = ctx().beam_select(logits, scores, k, done=done, eos=eos, **kw)
    torch.cuda.synchronize()
    assert torch.equal(got[1].cpu(), ref[1]) and torch.equal(got[2].cpu(), ref[2])
    # the score rounded once; lse off by the exponentials' arguments (2^-24 of up to 2^7 where they count), functions
    # (2 units) and the sums of 32 terms, which is 2^-18 of a share that adds up to one
    inside(got[0].cpu(), ref[0], ref[0].abs().nan_to_num(0, 0, 0) * F * 1.01 + 34 * F * 4)
    return got


def logits_of(batch, beams, vocab, dtype, seed=0, scale=3.0):
    return randn(batch, beams, vocab, dtype=dtype, seed=seed, scale=scale)


def scores_of(batch, beams, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    return -torch.rand(batch, beams, generator=g, device="cuda").mul(5).cumsum(1)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,lo,hi", [(8192, 100, 1100), (8192, 8000, 8192), (20000, 5, 17), (3000, 2040, 2100), (60000, 0, 3000)])
def test_beam_select_of_few_allowed_tokens(dtype, vocab, lo, hi):
    """A run of tokens, the others at -infinity: waves with and without numbers, fewer than k in all."""
    import torch
    x = torch.full((2, 3, vocab), -math.inf, dtype=tdt(dtype), device="cuda")
    x[..., lo:hi] = logits_of(2, 3, hi - lo, dtype, seed=lo)
    for k in (1, 7, 64, 65, 128):
        check_select(x, scores_of(2, 3), k)


SELECT = [(1, 1, 255, 100), (2, 2, 849, 128), (1, 3, 300, 64), (1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 10), (1, 4, 2048, 4), (1, 4, 2049, 8), (3, 2, 8191, 64), (1, 1, 50001, 128),
          (2, 5, 30000, 10), (2, 64, 1000, 128), (1, 7, 8, 56), (64, 8, 9001, 16), (3, 1, 300, 1), (1, 2, 260000, 100), (33, 16, 8200, 32)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("batch,beams,vocab,k", SELECT)
def test_beam_select(dtype, batch, beams, vocab, k):
    import torch
    x, s = logits_of(batch, beams, vocab, dtype, seed=vocab), scores_of(batch, beams, seed=k)
    check_select(x, s, k)
    g = torch.Generator(device="cuda").manual_seed(7)
    done = torch.rand(batch, beams, generator=g, device="cuda") < 0.4
    check_select(x, s, k, done=done, eos=vocab // 2)
    check_select(x, s, k, done=done.to(torch.uint8), eos=0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,rows", [(5000, 3), (17000, 3), (9000, 300)])
def test_beam_select_of_equal_and_ordered_logits(dtype, vocab, rows):
    """Far more logits reach the threshold than are kept: all equal, few levels, sorted both ways."""
    import torch
    t = torch.arange(vocab, device="cuda", dtype=torch.float32)
    for x in (torch.zeros(vocab, device="cuda"), (t * 7919 % 3), t / vocab, -t / vocab, (t % 40) - (t // 4000)):
        x = x.to(tdt(dtype)).expand(1, rows if rows < 10 else 4, vocab).repeat(1 if rows < 10 else rows // 4, 1, 1).contiguous()
        s = torch.zeros(x.shape[:2], device="cuda")
        for k in (1, 4, 33, 128):
            check_select(x, s, k)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_beam_select_of_what_is_no_number(dtype):
    """Forbidden tokens, beams that are not in use, infinities and NaN: -infinity, by place, behind all others."""
    import torch
    x, s = logits_of(2, 4, 6000, dtype, seed=3), scores_of(2, 4)
    x[0, 0, 7], x[0, 1, 5999] = math.nan, math.inf
    x[0, 2] = -math.inf
    x[0, 3, 3:] = -math.inf                     # three candidates in all
    x[1, 0, ::2] = -math.inf
    s[1, 1], s[1, 2], s[1, 3] = -math.inf, math.nan, math.inf
    check_select(x, s, 9)
    check_select(x, s, 128)
    s[:] = -math.inf
    got = check_select(x, s, 64)
    assert torch.all(got[0] == -math.inf) and got[2][0].tolist() == list(range(64))
    done = torch.ones(2, 4, device="cuda", dtype=torch.uint8)
    s = scores_of(2, 4)
    got = check_select(x, s, 6, done=done, eos=17)
    assert got[2][0].tolist()[:4] == [17] * 4
    first = torch.full((2, 4), -math.inf, device="cuda")      # the first step: one beam
    first[:, 0] = 0
    check_select(logits_of(2, 4, 6000, dtype, seed=5), first, 8)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_beam_select_of_masks_at_the_end_of_the_range(dtype):
    """Tokens masked by the type's lowest number are candidates like others, rows of nothing else too."""
    import torch
    low = torch.finfo(tdt(dtype)).min
    x, s = logits_of(2, 3, 5000, dtype, seed=3), scores_of(2, 3)
    x[0, 0, 4:] = low
    x[0, 1] = low
    x[0, 2, ::2] = low
    x[1] = -low
    check_select(x, s, 12)
    x[:] = low
    x[0, 1, 77] = 0
    check_select(x, s, 12)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("far", [1e5, 2e6, 1e8, 1e9, 4e9, 1e10, 1e11, 1e20, 9e29])
@pytest.mark.parametrize("batch,beams,vocab", [(2, 3, 5000), (75, 4, 17000)])
def test_beam_select_of_masks_far_from_zero(dtype, far, batch, beams, vocab):
    """Chunks of nothing but tokens masked by a large negative number, beams of nothing else, tokens forced by a large
    positive one: the sums' terms are in range wherever the chunk's largest logit lies."""
    import torch
    x, s = logits_of(batch, beams, vocab, dtype, seed=11), scores_of(batch, beams, seed=12)
    x[0, 0, vocab // 3:] = -far                  # whole chunks beside ordinary logits
    x[0, 1] = -far                               # nothing else
    x[0, 2, 9:] = -far
    x[1, 0, vocab - 5] = far                     # forced: the only one of its beam that counts
    x[1, 1] = far
    x[1, 2, ::2] = -far
    for k in (1, 8, 128):
        ref = select_ref(x, s, k)
        got = ctx().beam_select(x, s, k)
        torch.cuda.synchronize()
        assert torch.equal(got[1].cpu(), ref[1]) and torch.equal(got[2].cpu(), ref[2])
        # as check_select, and lse in 64 bits on either side: two roundings here and one there, each by 2^-53 of it
        lse = torch.logsumexp(x.double().cpu(), 2).abs().gather(1, ref[1].long())
        inside(got[0].cpu(), ref[0], ref[0].abs().nan_to_num(0, 0, 0) * F * 1.01 + 34 * F * 4 + lse * 2.0 ** -51)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_beam_select_of_beams_with_like_scores(dtype):
    """Many beams and chunks of which any may hold the best: far more entries reach the first threshold than are kept."""
    import torch
    for beams, vocab, k in ((26, 60405, 26), (64, 30000, 128), (40, 9000, 60)):
        x, s = logits_of(2, beams, vocab, dtype, seed=beams, scale=2.0), scores_of(2, beams) * 1e-3
        check_select(x, s, k)
        check_select(x.round(), torch.zeros_like(s), k)


def test_beam_select_equal_beams():
    """The same logits and score in every beam: equal candidates by the lowest beam."""
    x = logits_of(2, 1, 3000, "f32", seed=9).expand(2, 6, 3000).contiguous()
    got = check_select(x, scores_of(2, 1).expand(2, 6).contiguous(), 13)
    assert got[1][0].tolist()[:6] == list(range(6))


def test_beam_select_rows_of_any_alignment():
    import torch
    for dtype in ("bf16", "f32"):
        for pad, lead in ((1, 1), (3, 0), (8, 5)):
            buf = randn(2 * 3 * (2500 + pad) + lead, dtype=dtype, seed=pad, scale=3.0)
            x = buf[lead:].as_strided((2, 3, 2500), (3 * (2500 + pad), 2500 + pad, 1))
            check_select(x, scores_of(2, 3), 5)
        buf = randn(2, 4, 2500, dtype=dtype)
        with pytest.raises(ValueError, match="stride"):
            ctx().beam_select(buf[:, :3], scores_of(2, 3), 5)


def test_beam_select_workspace_outputs_and_graph():
    import torch
    x, s = logits_of(3, 4, 40000, "bf16", seed=1), scores_of(3, 4)
    want = check_select(x, s, 8)
    need = vrs.lib().vrs_beam_select_workspace_size(vrs._BEAM(3, 4, 40000, 8, vrs.BF16, -1, 40000))
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    outs = tuple(torch.full_like(t, 9) for t in want)
    call = lambda: ctx().beam_select(x, s, 8, outs=outs, workspace=ws)   # noqa: E731
    assert call() is outs
    with pytest.raises(vrs.VrsError):
        ctx().beam_select(x, s, 8, workspace=ws[:-16])
    for got in replayed(call, outs, lambda: [t.fill_(9) for t in outs]):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- beam search: the reordering --------------------------------------------------------


def reorder_ref(state, parents, lens):
    out = state.clone()
    batch, beams = parents.shape
    P = parents.tolist()
    L = None if lens is None else lens.flatten().tolist()
    for b in range(batch):
        for i, p in enumerate(P[b]):
            if 0 <= p < beams:
                n = state.shape[2] if L is None else max(0, min(L[b * beams + p], state.shape[2]))
                out[:, b * beams + i, :n] = state[:, b * beams + p, :n]
    return out


@pytest.mark.parametrize("layers,batch,beams,rows,row,dtype", [
    (1, 1, 1, 3, (8,), "f32"), (2, 3, 4, 10, (2, 64), "bf16"), (3, 2, 5, 33, (7,), "bf16"), (1, 2, 16, 40, (24,), "f32"),
    (2, 1, 17, 9, (8,), "bf16"), (1, 3, 64, 20, (16,), "f32"), (1, 2, 64, 300, (1,), "u8"), (4, 2, 8, 1, (), "i32"),
    (1, 5, 3, 100, (3,), "u8"), (2, 2, 2, 700, (128,), "bf16"),
])
def test_beam_reorder(layers, batch, beams, rows, row, dtype):
    """Any permutation and any repetition; slots of unequal lengths; parents that are none."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(beams * rows)
    dt = {"f32": torch.float32, "bf16": torch.bfloat16, "u8": torch.uint8, "i32": torch.int32}[dtype]
    for turn in range(5):
        state = torch.randint(0, 200, (layers, batch * beams, rows, *row), generator=g, device="cuda").to(dt)
        parents = torch.randint(0, beams, (batch, beams), generator=g, device="cuda", dtype=torch.int32)
        lens = torch.randint(-3, rows + 5, (batch * beams,), generator=g, device="cuda", dtype=torch.int32)
        if turn == 1:
            parents = torch.stack([torch.randperm(beams, generator=g, device="cuda") for _ in range(batch)]).int()
            lens = None
        if turn == 2:
            parents[:] = beams - 1
        if turn == 3:
            parents = torch.randint(-2, beams + 2, (batch, beams), generator=g, device="cuda", dtype=torch.int32)
            lens = lens.view(batch, beams)
        if turn == 4:
            parents = torch.arange(beams, device="cuda", dtype=torch.int32).expand(batch, beams).contiguous()
        want = reorder_ref(state, parents, lens)
        assert ctx().beam_reorder(state, parents, lens=lens) is state
        assert torch.equal(state, want)


def test_beam_reorder_strides():
    """Layers inside slots, rows apart, heads outside a slot's rows, addresses off 16 bytes: what lies between stays."""
    import torch
    for dtype, pad in ((torch.float32, 2), (torch.bfloat16, 3), (torch.uint8, 1)):
        buf = torch.randint(0, 200, (6, 3, 20, 8 + pad), device="cuda").to(dtype)       # slot, layer, row, element
        state = buf.transpose(0, 1)[:, :, :, pad:]
        parents, lens = i32([[2, 2, 0], [1, 0, 0]]), i32([20, 4, 7, 9, 0, 3])
        want_buf = buf.clone()
        want_buf.transpose(0, 1)[:, :, :, pad:] = reorder_ref(state, parents, lens)
        ctx().beam_reorder(state, parents, lens=lens)
        assert torch.equal(buf, want_buf)
    cache = torch.randn(6, 4, 20, 16, device="cuda")                                    # slot, head, row, element
    want = reorder_ref(cache.transpose(0, 1), parents, lens).transpose(0, 1).contiguous()
    ctx().beam_reorder(cache.transpose(0, 1), parents, lens=lens)
    assert torch.equal(cache, want)


def test_beam_reorder_graph():
    import torch
    state0 = torch.randn(2, 8, 30, 64, device="cuda")
    state = state0.clone()
    parents = i32([[3, 0, 0, 1], [0, 1, 2, 3]])
    want = reorder_ref(state, parents, None)
    for (got,) in replayed(lambda: ctx().beam_reorder(state, parents), [state], lambda: state.copy_(state0)):
        assert torch.equal(got, want)


# ---- attention that keys receive ---------------------------------------------------------

CASES = {
    "prompts": ([40, 130, 1, 65], [0, 0, 3, 10]),
    "tokens": ([1] * 6, [5, 0, 33, 64, 700, 200]),
    "mixed": ([3, 0, 130, 1, 64], [7, 5, 0, 2000, 61]),
    "short": ([5, 9, 0], [-3, -20, 4]),
    "many": ([1] * 80, [i % 40 for i in range(80)]),
    "few": ([8, 5], [300, 1000]),
}


def weights_case(case, lead=2, tail=3, hint=True):
    q_len, past = CASES[case] if isinstance(case, str) else case
    starts = [lead + sum(q_len[:i]) for i in range(len(q_len) + 1)]
    k_len = [max(0, a + b) for a, b in zip(q_len, past)]
    k_at = [int(x) for x in np.cumsum([1] + [n + 3 for n in k_len])]
    h = dict(max_q=max(q_len), max_k=max(k_len)) if hint else {}
    return starts, starts[-1] + tail, k_len, k_at, vrs.seqs(i32(starts), i32(k_at[:-1]), i32(k_len), **h)


def weights_ref(q, k, acc, starts, k_len, k_at, causal, scale, decay):
    import torch
    ref, tol = acc.double().clone(), torch.zeros(acc.shape, dtype=torch.float64, device=acc.device)
    H, KV, D = q.shape[1], k.shape[1], q.shape[2]
    for i, n in enumerate(k_len):
        a, b, at = starts[i], starts[i + 1], slice(k_at[i], k_at[i] + n)
        if n == 0:
            continue
        ref[:, at] = ref[:, at] * decay if decay else 0.0
        tol[:, at] = ref[:, at].abs() * 2 * F
        if a == b:
            continue
        Q = q[a:b].double().transpose(0, 1)
        K = k[at].double().repeat_interleave(H // KV, 1).transpose(0, 1)
        seen = torch.ones(b - a, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(n, device=q.device)[None] <= (n - (b - a) + torch.arange(b - a, device=q.device))[:, None]
        s = (Q @ K.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        w = torch.where(seen, torch.softmax(s, 2), 0.0)
        got = w.view(KV, H // KV, b - a, n).sum((1, 2))
        # scores off by e, which is 2 e of a weight with its sum's; float32 sums over the keys and over the rows
        big = (Q.abs() @ K.abs().transpose(1, 2) * scale).masked_fill(~seen, 0).nan_to_num(0, 0, 0).amax(2, keepdim=True)
        e = (D + 8) * F * big + 8 * F
        off = (w.nan_to_num(0) * (2 * e * 1.02 + (n + 70) * F)).view(KV, H // KV, b - a, n).sum((1, 2))
        ref[:, at] += got
        tol[:, at] += off + (got.nan_to_num(0) + ref[:, at].nan_to_num(0).abs()) * ((b - a) * H // KV + 4) * F
    return ref, tol


def check_weights(case, dtype="bf16", heads=4, kv=2, dim=64, causal=True, decay=1.0, scale=0.0, hint=True, seed=0, edit=None):
    import torch
    starts, rows, k_len, k_at, s = weights_case(case, hint=hint)
    q, k = randn(rows, heads, dim, dtype=dtype, seed=seed, scale=2), randn(k_at[-1] + 4, kv, dim, dtype=dtype, seed=seed + 1)
    acc = torch.rand(kv, k_at[-1] + 4, device="cuda")
    if edit:
        edit(q, k, acc, k_at, k_len)
    ref, tol = weights_ref(q, k, acc, starts, k_len, k_at, causal, scale or dim ** -0.5, decay)
    assert ctx().attention_weights(q, k, s, acc, decay=decay, causal=causal, scale=scale) is acc
    inside(acc, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (3, 3, 8), (8, 1, 128), (5, 1, 72)])
def test_attention_weights(dtype, causal, case, heads, kv, dim):
    check_weights(case, dtype, heads, kv, dim, causal, decay=1.0 if causal else 0.5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 64, 127, 128, 129, 257, 4000])
def test_attention_weights_lengths(dtype, n):
    check_weights(([n], [0]), dtype, 4, 2, 64, seed=n)
    check_weights(([1, 1], [n - 1, n]), dtype, 8, 2, 128, seed=n)
    check_weights(([60, 1], [n, n]), dtype, 4, 1, 72, seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_weights_decay_and_what_is_not_finite(dtype):
    """decay 0 does not read acc; a key behind the last, or one that a query does not see, touches nothing; a query
    all of whose keys score -infinity gives NaN to those it sees."""
    def edit(q, k, acc, k_at, k_len):
        acc[:, :k_at[-1]] = math.nan
        for i, n in enumerate(k_len):
            k[k_at[i] + n] = math.nan
    for case in ("prompts", "tokens", "few"):
        check_weights(case, dtype, decay=0.0, edit=edit)

    def lost(q, k, acc, k_at, k_len):
        q[:], k[:] = 0, 0
        q[..., 0] = 1
        k[k_at[0]:k_at[0] + 3, 0, 0] = -math.inf
    for q_len, past in ((4, 0), (40, 0), (1, 2)):
        check_weights(([q_len, 3], [past, 4]), dtype, 4, 2, 64, edit=lost)


def test_attention_weights_hints_choose_kernels_only():
    import torch
    for case in ("prompts", "tokens", "few", "mixed"):
        starts, rows, k_len, k_at, s = weights_case(case)
        q, k = randn(rows, 4, 64, seed=1, scale=2), randn(k_at[-1] + 4, 2, 64, seed=2)
        acc = torch.rand(2, k_at[-1] + 4, device="cuda")
        ref, tol = weights_ref(q, k, acc, starts, k_len, k_at, True, 0.125, 1.0)
        for max_q, max_k in ((0, 0), (1, 1), (1, 0), (1, 10), (5, 4000), (1 << 30, 1 << 30), (64, 1)):
            s.max_q, s.max_k = max_q, max_k
            inside(ctx().attention_weights(q, k, s, acc.clone()), ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv", [(7, 1), (66, 1), (12, 4), (40, 8)])
def test_attention_weights_groups_of_any_size(dtype, heads, kv):
    """Row tiles that end inside a query, groups larger than a tile; parts of rows and of keys."""
    check_weights(([130, 3, 40], [0, 500, 7]), dtype, heads, kv, 64, True)
    check_weights(([33], [3000]), dtype, heads, kv, 72, True, seed=heads)
    check_weights(([600, 500], [0, 0]), dtype, heads, kv, 32, False, seed=kv)


def test_attention_weights_large_and_far_scores():
    for dtype in ("bf16", "f32"):
        check_weights("few", dtype, scale=3.0)
        check_weights("prompts", dtype, scale=3.0)
        check_weights("tokens", dtype, scale=1e-4)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len,past", [([1, 1], [60, 700]), ([60, 3], [0, 40]), ([50], [2000])])
def test_attention_weights_of_scores_far_from_zero(dtype, q_len, past):
    """Scores of 2^34, exact in either type: those keys share each query's weight evenly, the others get none."""
    import torch
    starts, rows, k_len, k_at, s = weights_case((q_len, past))
    q = torch.zeros(rows, 4, 64, dtype=tdt(dtype), device="cuda")
    k = torch.zeros(k_at[-1] + 4, 2, 64, dtype=tdt(dtype), device="cuda")
    q[..., 0] = 2.0 ** 17
    acc = torch.zeros(2, k_at[-1] + 4, device="cuda")
    ref = acc.double()
    for i, (n, m) in enumerate(zip(k_len, q_len)):
        large = [j for j in (0, 7, 33, 59, n - 1) if j < n]
        k[[k_at[i] + j for j in large], :, 0] = 2.0 ** 17
        for j in range(m):
            seen = [x for x in set(large) if x <= n - m + j]
            for x in seen:
                ref[:, k_at[i] + x] += 2 / len(seen)           # two heads of a key head
    ctx().attention_weights(q, k, s, acc, scale=1.0)
    inside(acc, ref, ref * 200 * F)


def test_attention_weights_strides_workspace_and_graph():
    """acc with the heads inside its rows, views, a workspace full of NaN, replays."""
    import torch
    for case in ("prompts", "tokens"):
        starts, rows, k_len, k_at, s = weights_case(case)
        n_k = k_at[-1] + 4
        q, k = randn(rows, 6, 64, seed=1, scale=2)[:, 1:5], randn(n_k, 4, 64, seed=2)[:, ::2]
        buf = torch.rand(n_k, 3, device="cuda")
        buf0, acc = buf.clone(), buf.t()[1:]
        ref, tol = weights_ref(q, k, acc, starts, k_len, k_at, True, 0.125, 0.75)
        d = vrs._WEIGHTS(rows, n_k, 4, 2, 64, vrs.BF16, 1, 0.0, 0.75, 6 * 64, 64, 4 * 64, 128, 3, 1)
        need = vrs.lib().vrs_attention_weights_workspace_size(d, s.address)
        ws = torch.full((need // 4,), math.nan, device="cuda").view(torch.uint8)
        call = lambda: ctx().attention_weights(q, k, s, acc, decay=0.75, workspace=ws)   # noqa: E731
        call()
        inside(acc, ref, tol)
        want = acc.clone()
        assert torch.equal(buf[:, 0], buf0[:, 0])
        with pytest.raises(vrs.VrsError):
            ctx().attention_weights(q, k, s, acc, workspace=ws[:-16])
        for (got,) in replayed(call, [buf], lambda: buf.copy_(buf0)):
            assert torch.equal(got.t()[1:], want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_weights_of_rows_whose_keys_are_in_parts(dtype):
    """A workspace full of NaN, rows of no sequence, replays that follow the lengths."""
    import torch
    case = ([40, 0, 70, 1], [3000, 9, 500, 200])
    starts, rows, k_len, k_at, s = weights_case(case)
    q, k = randn(rows, 4, 64, dtype=dtype, seed=1, scale=2), randn(k_at[-1] + 4, 2, 64, dtype=dtype, seed=2)
    acc0 = torch.rand(2, k_at[-1] + 4, device="cuda")
    d = vrs._WEIGHTS(rows, k.shape[0], 4, 2, 64, vrs.F32 if dtype == "f32" else vrs.BF16, 1, 0.0, 0.5, 256, 64, 128, 64, 1, k.shape[0])
    ws = torch.full((vrs.lib().vrs_attention_weights_workspace_size(d, s.address) // 4,), math.nan, device="cuda").view(torch.uint8)
    assert ws.numel() >= 2 * 8 * rows * 4                   # two parts at least
    acc = acc0.clone()
    call = lambda: ctx().attention_weights(q, k, s, acc, decay=0.5, workspace=ws)   # noqa: E731
    ref, tol = weights_ref(q, k, acc0, starts, k_len, k_at, True, 0.125, 0.5)
    call()
    inside(acc, ref, tol)
    want = acc.clone()
    for (got,) in replayed(call, [acc], lambda: acc.copy_(acc0)):
        assert torch.equal(got, want)
    k_len[0] = 41                                           # the captured call would see these
    s.tensors[2].copy_(i32(k_len))
    ref, tol = weights_ref(q, k, acc0, starts, k_len, k_at, True, 0.125, 0.5)
    for (got,) in replayed(call, [acc], lambda: acc.copy_(acc0)):
        inside(got, ref, tol)


def test_attention_weights_writes_no_key_outside():
    import torch
    buf = torch.full((1, 60), 7.0, device="cuda")
    q, k = randn(6, 1, 64, seed=1), randn(40, 1, 64, seed=2)
    for q_start in ([0, 2, 4, 900], [-5, 1, 3, 4]):
        for hint in (dict(max_q=1, max_k=5), dict(max_q=100)):
            s = vrs.seqs(i32(q_start), i32([-3, 30, 38]), i32([4, 100, 1 << 30]), **hint)
            ctx().attention_weights(q, k, s, buf[:, 10:50])
            torch.cuda.synchronize()
            assert torch.all(buf[:, :10] == 7) and torch.all(buf[:, 50:] == 7) and torch.all(buf[:, 10:40] == 7)


# ---- eviction ------------------------------------------------------------------------------


def evict_ref(k, v, acc, k_at, k_len, budget, first, recent, outs, o_at):
    import torch
    ko, vo, ao = (t.clone() for t in outs)
    kept = torch.full((len(k_len), k.shape[1], budget), -1, dtype=torch.int32, device=k.device)
    for i, n in enumerate(k_len):
        left = min(n, budget)
        for h in range(k.shape[1]):
            a = acc[h, k_at[i]:k_at[i] + n].double().cpu().tolist()
            must = [j for j in range(n) if j < first or j >= n - recent] if n > budget else list(range(n))
            rest = sorted(set(range(n)) - set(must), key=lambda j: (-(math.inf if a[j] != a[j] else a[j]), 0 if a[j] != a[j] else 1, j))
            keep = sorted(must + rest[:left - len(must)])
            kept[i, h, :left] = torch.tensor(keep, dtype=torch.int32, device=k.device)
            src = torch.tensor(keep, dtype=torch.long, device=k.device) + k_at[i]
            to = slice(o_at[i], o_at[i] + left)
            ko[to, h], vo[to, h], ao[h, to] = k[src, h], v[src, h], acc[h, src]
    return ko, vo, ao, kept


def bits(t):
    import torch
    return t.contiguous().view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def check_evict(k_len, budget, first=0, recent=0, dtype="bf16", kv=2, dim=64, inplace=True, acc=None, seed=0, edit=None):
    import torch
    n = len(k_len)
    k_at = [int(x) for x in np.cumsum([1] + [max(m, budget) + 2 for m in k_len])]
    rows = k_at[-1] + 3
    k, v = randn(rows, kv, dim, dtype=dtype, seed=seed), randn(rows, kv, dim, dtype=dtype, seed=seed + 1)
    if acc is None:
        g = torch.Generator(device="cuda").manual_seed(seed)
        acc = torch.rand(kv, rows, generator=g, device="cuda")
    if edit:
        edit(acc, k_at)
    outs, o_at, o_start = (k, v, acc), k_at, None
    if not inplace:
        o_at = [int(x) for x in np.cumsum([2] + [budget + 1] * n)]
        outs = (torch.full((o_at[-1] + 4, kv, dim), 5.0, dtype=tdt(dtype), device="cuda"),
                torch.full((o_at[-1] + 4, kv, dim), 6.0, dtype=tdt(dtype), device="cuda"), torch.full((kv, o_at[-1] + 4), 7.0, device="cuda"))
        o_start = i32(o_at[:-1])
    ref = evict_ref(k, v, acc, k_at, k_len, budget, first, recent, outs, o_at)
    lens = i32(k_len)
    kept, len_out = ctx().cache_evict(k, v, acc, i32(k_at[:-1]), lens, budget, first=first, recent=recent, max_k=max(k_len),
                                      k_out=outs[0], v_out=outs[1], acc_out=outs[2], out_start=o_start,
                                      len_out=lens if inplace else None)
    torch.cuda.synchronize()
    assert torch.equal(kept, ref[3])
    assert len_out.tolist() == [min(m, budget) for m in k_len]
    for got, want in zip(outs, ref):
        assert torch.equal(bits(got), bits(want))


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 72), ("bf16", 6), ("bf16", 7), ("f32", 1)])
@pytest.mark.parametrize("inplace", [True, False])
@pytest.mark.parametrize("k_len,budget,first,recent", [
    ([1], 1, 0, 0), ([0, 2, 1], 1, 0, 1), ([700, 64, 63, 65, 0], 64, 4, 16), ([1500, 900], 512, 0, 0), ([100, 1100], 1024, 1000, 24),
    ([3000], 17, 1, 15), ([1023, 1024, 1025, 2049], 1000, 4, 100), ([50] * 70, 20, 2, 3),
])
def test_cache_evict(dtype, dim, inplace, k_len, budget, first, recent):
    check_evict(k_len, budget, first, recent, dtype, 2, dim, inplace)


@pytest.mark.parametrize("inplace", [True, False])
def test_cache_evict_long(inplace):
    """More keys than the choice holds in registers (16384)."""
    check_evict([16384, 16385, 40000], 9000, 4, 500, "bf16", 1, 8, inplace)
    check_evict([20000], 19999, 0, 0, "bf16", 1, 8, inplace)


def test_cache_evict_hint_chooses_kernels_only():
    import torch
    for k_len, budget in (([9000, 20, 4097], 700), ([300, 90], 64)):
        k_at, rows = [0, 9001, 9030][:len(k_len)], 14000
        k, v, acc = randn(rows, 2, 64, seed=1), randn(rows, 2, 64, seed=2), torch.rand(2, rows, device="cuda")
        ref = evict_ref(k, v, acc, k_at, k_len, budget, 2, 30, (k, v, acc), k_at)
        for hint in (0, 1, 4096, 4097, (1 << 31) - 1):
            outs = [t.clone() for t in (k, v, acc)]
            kept, _ = ctx().cache_evict(*outs, i32(k_at), i32(k_len), budget, first=2, recent=30, max_k=hint)
            assert all(torch.equal(a, b) for a, b in zip((*outs, kept), ref)), hint


def test_cache_evict_equal_and_odd_values():
    """Equal weights: the earliest; zeros of either sign alike; NaN above infinity; negative ones."""
    import torch

    def equal(acc, k_at):
        acc[:] = 0.5

    def levels(acc, k_at):
        acc[:] = (torch.arange(acc.shape[1], device="cuda") * 7919 % 5) / 4

    def odd(acc, k_at):
        acc[:, ::3] = 0.0
        acc[:, 1::3] = -0.0
        acc[:, ::11] = math.nan
        acc[:, 4::13] = math.inf
        acc[:, 5::17] = -math.inf
        acc[:, 6::19] = -2.5

    def tiny(acc, k_at):
        acc *= 1e-44
    for edit in (equal, levels, odd, tiny):
        for budget, first, recent in ((10, 0, 0), (300, 4, 30), (1100, 1, 0)):
            for inplace in (True, False):
                check_evict([1500, 40, 1100, 1101], budget, first, recent, edit=edit, inplace=inplace)


def test_cache_evict_strides():
    """Caches with the heads outside a sequence's rows, acc with the heads inside: the bits of the plain layout."""
    import torch
    n, kv, room, dim = 3, 2, 90, 64
    lens = i32([90, 20, 61])
    kc, vc = randn(n, kv, room, dim, seed=2), randn(n, kv, room, dim, seed=3)
    acc = torch.rand(n, kv, room, device="cuda")
    plain = [t.transpose(1, 2).reshape(n * room, kv, dim).clone() for t in (kc, vc)]
    pacc = acc.transpose(0, 1).reshape(kv, n * room).clone()
    kept, left = ctx().cache_evict(*plain, pacc, i32([0, room, 2 * room]), lens, 40, first=2, recent=10)
    rows = (n * kv - (kv - 1)) * room
    view = [t.as_strided((rows, kv, dim), (dim, room * dim, 1)) for t in (kc, vc)]
    vacc = acc.as_strided((kv, rows), (room, 1))
    kept2, left2 = ctx().cache_evict(*view, vacc, i32([i * kv * room for i in range(n)]), lens, 40, first=2, recent=10)
    assert torch.equal(kept, kept2) and torch.equal(left, left2)
    for a, b in zip((kc, vc), plain):
        assert torch.equal(a, b.view(n, room, kv, dim).transpose(1, 2))
    assert torch.equal(acc, pacc.view(kv, n, room).transpose(0, 1))
    inner = torch.rand(n * room, kv + 1, device="cuda")
    k, v = randn(n * room, kv, dim, seed=5), randn(n * room, kv, dim, seed=6)
    outer = inner[:, 1:].t().contiguous()
    k2, v2 = k.clone(), v.clone()
    a = ctx().cache_evict(k, v, inner[:, 1:].t(), i32([0, room, 2 * room]), lens, 33)
    b = ctx().cache_evict(k2, v2, outer, i32([0, room, 2 * room]), lens, 33)
    assert torch.equal(a[0], b[0]) and torch.equal(k, k2) and torch.equal(v, v2) and torch.equal(inner[:, 1:].t(), outer)


def test_cache_evict_writes_no_row_outside():
    """Starts and lengths that do not fit the buffers are cut off."""
    import torch
    k, v = randn(40, 1, 64, seed=1), randn(40, 1, 64, seed=2)
    acc = torch.rand(1, 40, device="cuda")
    big = [torch.full((40, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    acco = torch.full((1, 40), 7.0, device="cuda")
    kept, lens = ctx().cache_evict(k, v, acc, i32([-1, 35, 100, 3]), i32([5, 1 << 30, 3, -2]), 8, out_start=i32([0, 7, 2, 2]),
                                   k_out=big[0][10:20], v_out=big[1][10:20], acc_out=acco[:, 10:20])
    torch.cuda.synchronize()
    assert lens.tolist() == [0, 5, 0, 0] and kept[1, 0].tolist() == [0, 1, 2, 3, 4, -1, -1, -1]
    for t in (*big, acco.t()[:, :, None]):
        assert torch.all(t[:17] == 7) and torch.all(t[20:] == 7)
    assert torch.equal(big[0][17:20], k[35:38])


def test_cache_evict_graph():
    import torch
    k0, v0, acc0 = randn(3000, 2, 64, seed=1), randn(3000, 2, 64, seed=2), torch.rand(2, 3000, device="cuda")
    at, lens0 = i32([0, 1500]), i32([1500, 1200])
    k, v, acc, lens = k0.clone(), v0.clone(), acc0.clone(), lens0.clone()
    kept = torch.zeros(2, 2, 300, dtype=torch.int32, device="cuda")

    def reset():
        for a, b in ((k, k0), (v, v0), (acc, acc0), (lens, lens0)):
            a.copy_(b)
    want = [*evict_ref(k, v, acc, [0, 1500], [1500, 1200], 300, 4, 50, (k, v, acc), [0, 1500]), i32([300, 300])]
    for got in replayed(lambda: ctx().cache_evict(k, v, acc, at, lens, 300, first=4, recent=50, len_out=lens, kept=kept),
                        [k, v, acc, kept, lens], reset):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- together --------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_beam_search_over_an_evicted_prompt(dtype):
    """Two prompts are weighed and cut to their budget; four beams of each go on from what is left: attention over
    the shared prefix and the own keys, a selection, the reordering of keys, values, lengths and tokens.  Every
    operator's result is checked on the state that it met; then a captured step has the eager one's bits."""
    import torch
    heads, kv, dim, vocab, beams, steps, budget = 4, 2, 64, 500, 4, 4, 48
    n = 2 * beams
    prompt, p_at = [90, 130], [0, 130]
    own0, room = 260, steps + 2
    k, v = randn(own0 + n * room, kv, dim, dtype=dtype, seed=1), randn(own0 + n * room, kv, dim, dtype=dtype, seed=2)
    q0 = randn(sum(prompt), heads, dim, dtype=dtype, seed=3, scale=2)
    acc = torch.zeros(kv, k.shape[0], device="cuda")
    s0 = vrs.seqs(i32([0, 90, 220]), i32(p_at), i32(prompt), max_q=130, max_k=130)
    ref, tol = weights_ref(q0, k, acc, [0, 90, 220], prompt, p_at, True, dim ** -0.5, 1.0)
    ctx().attention_weights(q0, k, s0, acc)
    inside(acc, ref, tol)
    p_len = i32(prompt)
    want = evict_ref(k, v, acc, p_at, prompt, budget, 4, 8, (k, v, acc), p_at)
    kept, _ = ctx().cache_evict(k, v, acc, i32(p_at), p_len, budget, first=4, recent=8, len_out=p_len)
    assert torch.equal(kept, want[3]) and torch.equal(k, want[0]) and torch.equal(v, want[1]) and p_len.tolist() == [budget] * 2

    embed, w_out = randn(vocab, heads + 2 * kv, dim, dtype=dtype, seed=4), randn(heads * dim, vocab, dtype="f32", seed=5, scale=0.3)
    k_start, k_len = i32([own0 + i * room for i in range(n)]), i32([0] * n)
    seqs = vrs.seqs(i32(list(range(n + 1))), k_start, k_len, max_q=1, max_k=room)
    pre = vrs.prefixes(i32([0, beams, n]), i32(p_at), p_len, max_rows=beams, max_k=budget)
    token = torch.zeros(2, beams, dtype=torch.int32, device="cuda")
    score = torch.full((2, beams), -math.inf, device="cuda")
    score[:, 0] = 0
    done = torch.zeros(2, beams, dtype=torch.bool, device="cuda")
    text = torch.zeros(1, n, steps + 4, dtype=torch.int32, device="cuda")
    freq = vrs.rope_freqs(dim // 2).cuda()
    own = [t[own0:].view(n, room, kv * dim)[None] for t in (k, v)]
    out = torch.empty(n, heads, dim, dtype=tdt(dtype), device="cuda")
    picks = (torch.empty_like(score), torch.empty_like(token), torch.empty_like(token))
    behind = torch.repeat_interleave(i32(prompt), beams) - 1
    trace = {}

    def step():
        k_len.add_(1)
        qkv = embed[token.flatten().long()]
        pos = behind + k_len              # positions go on from the whole prompt's
        q, _ = ctx().rope(qkv[:, :heads], qkv[:, heads:heads + kv], freq, seqs=seqs, positions=pos, k_out=k, v=qkv[:, heads + kv:], v_out=v)
        ctx().prefix_attention(q, k, v, seqs, pre, out=out)
        logits = (out.float().view(n, -1) @ w_out).view(2, beams, vocab)
        trace.update(q=q, logits=logits, score=score.clone(), done=done.clone(), k=k.clone(), v=v.clone(), text=text.clone())
        ctx().beam_select(logits, score, beams, done=done, eos=7, outs=picks)
        for t in own:
            ctx().beam_reorder(t, picks[1], lens=k_len)
        ctx().beam_reorder(text, picks[1])
        text.scatter_(2, k_len.long().view(1, n, 1), picks[2].view(1, n, 1))
        done.copy_(done.gather(1, picks[1].long()) | (picks[2] == 7))
        score.copy_(picks[0])
        token.copy_(picks[2])

    states = (k, v, k_len, token, score, done, text)
    for i in range(steps):
        if i == steps - 1:
            before = [t.clone() for t in states]
        step()
        b = dict(starts=list(range(n + 1)), k_len=[i + 1] * n, k_at=k_start.tolist(), group=[0] * beams + [1] * beams, p_at=p_at,
                 prefix=[budget] * 2)
        ref, tol = prefix_ref(b, trace["q"], trace["k"], trace["v"], True, dim ** -0.5, out, dtype)
        inside(out, ref, tol)
        rs, rp, rt = select_ref(trace["logits"], trace["score"], beams, trace["done"], 7)
        assert torch.equal(picks[1].cpu(), rp) and torch.equal(picks[2].cpu(), rt)
        inside(picks[0].cpu(), rs, rs.abs().nan_to_num(0, 0, 0) * F * 1.01 + 34 * F * 4)
        for now, was in ((k, trace["k"]), (v, trace["v"])):
            w = was.clone()
            w[own0:] = reorder_ref(was[own0:].view(n, room, -1)[None], picks[1], k_len)[0].reshape(-1, kv, dim)
            assert torch.equal(now, w)
    after = [t.clone() for t in states]

    def reset():
        for t, b0 in zip(states, before):
            t.copy_(b0)
    reset()
    for got in replayed(step, states, reset):
        assert all(torch.equal(a, b0) for a, b0 in zip(got, after))


def test_calls_on_two_streams_at_once():
    """Each operator on two streams that are not the current one, with workspaces of their own: the bits of calls one
    after another."""
    import torch
    b = build("group")
    q, k, v, out = prefix_inputs(b, "bf16", 8, 2, 64)
    x, s = logits_of(4, 8, 60000, "bf16", seed=2), scores_of(4, 8)
    state0, parents = torch.randn(3, 32, 50, 64, device="cuda"), torch.randint(0, 8, (4, 8), device="cuda", dtype=torch.int32)
    acc0 = torch.rand(2, b["k_rows"], device="cuda")
    at, lens = i32(b["k_at"][:-1]), i32(b["k_len"])

    def run(stream):
        state, acc, kk, vv = state0.clone(), acc0.clone(), k.clone(), v.clone()
        torch.cuda.synchronize()
        got = [ctx().prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=out.clone(), stream=stream),
               *ctx().beam_select(x, s, 8, stream=stream), ctx().beam_reorder(state, parents, stream=stream),
               ctx().attention_weights(q, k, b["seqs"], acc, stream=stream),
               *ctx().cache_evict(kk, vv, acc0.clone(), at, lens, 2, stream=stream), kk, vv]
        return got
    want = run(None)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [run(t.cuda_stream) for t in streams]
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(bits(a), bits(c)) for a, c in zip(g, want))


def test_calls_that_overlap_on_two_streams():
    """Two streams that run the operators at once, each in another order and with inputs and workspaces of its own: the
    bits of calls one after another.  All inputs are there before the first call, and nothing waits until the last."""
    import torch
    b = build(([1] * 48, [200 + i for i in range(48)], [0, 24, 48], [3000, 1700]))
    q, k, v, out = prefix_inputs(b, "bf16", 32, 8, 128)
    x, s = logits_of(8, 8, 60000, "bf16", seed=2), scores_of(8, 8)
    state0, parents = torch.randn(6, 64, 50, 128, device="cuda"), torch.randint(0, 8, (8, 8), device="cuda", dtype=torch.int32)
    acc0 = torch.rand(8, b["k_rows"], device="cuda")
    at, lens = i32(b["k_at"][:-1]), i32(b["k_len"])

    def jobs(stream):
        state, acc, kk, vv, aa, o = state0.clone(), acc0.clone(), k.clone(), v.clone(), acc0.clone(), out.clone()
        c = ctx()
        return [lambda: [c.prefix_attention(q, k, v, b["seqs"], b["prefixes"], out=o, stream=stream)],
                lambda: [*c.beam_select(x, s, 8, stream=stream)],
                lambda: [c.beam_reorder(state, parents, stream=stream)],
                lambda: [c.attention_weights(q, k, b["seqs"], acc, stream=stream)],
                lambda: [*c.cache_evict(kk, vv, aa, at, lens, 150, first=4, recent=20, stream=stream), kk, vv, aa]]
    want = [call() for call in jobs(None)]
    streams, turns = [torch.cuda.Stream() for _ in range(2)], 5
    calls = [[jobs(t.cuda_stream) for t in streams] for _ in range(turns)]
    torch.cuda.synchronize()
    got = []
    for turn in calls:
        for i in range(len(want)):
            for j, mine in enumerate(turn):
                n = (i + 2 * j) % len(want)
                got.append((n, mine[n]()))
    torch.cuda.synchronize()
    for n, outs in got:
        assert all(torch.equal(bits(a), bits(c)) for a, c in zip(outs, want[n])), n


@pytest.mark.parametrize("case", [([2] * 210, [3 + i % 40 for i in range(210)], [3 * i for i in range(71)], [5 * i for i in range(70)]),
                                  ([40] * 70, [i % 9 for i in range(70)], [0, 1, 30, 70], [300, 0, 41])])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prefix_attention_of_many_groups_of_many_rows(dtype, case):
    """Over 64 groups, or sequences, whose row tiles are found by a search."""
    check_prefix(case, dtype, 8, 1, 64)
    check_prefix(case, dtype, 8, 1, 64, hint=False)


def test_empty_batches_and_caches():
    """No keys, no sequences, no requests, no layers: results of nothing, and nothing else is touched."""
    import torch
    e = lambda *shape, dt=torch.bfloat16: torch.empty(shape, dtype=dt, device="cuda")      # noqa: E731
    q = randn(6, 4, 64, seed=1)
    for q_start in ([0, 1, 2], [0, 2, 6], [0, 0, 0]):
        for prefix in (([0, 2], [0], [5]), ([0, 0, 2], [0, 3], [0, 9]), ([0], [], [])):
            out = torch.full((6, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
            s = vrs.seqs(i32(q_start), i32([0, 0]), i32([0, 4]))
            ctx().prefix_attention(q, e(0, 2, 64), e(0, 2, 64), s, vrs.prefixes(*map(i32, prefix)), out=out)
            assert not out[:q_start[-1]].any() and torch.all(out[q_start[-1]:] == 5)
    s = vrs.seqs(i32([0]), i32([]), i32([]))
    k = randn(9, 2, 64, seed=2)
    acc = torch.full((2, 9), 3.0, device="cuda")
    assert ctx().prefix_attention(q, k, k, s, vrs.prefixes(i32([0, 0]), i32([0]), i32([9]))).shape == q.shape
    ctx().attention_weights(q, k, s, acc)
    ctx().attention_weights(q, e(0, 2, 64), vrs.seqs(i32([0, 6]), i32([0]), i32([3])), e(2, 0, dt=torch.float32))
    assert torch.all(acc == 3)
    ctx().attention_weights(e(0, 4, 64), k, vrs.seqs(i32([0, 0]), i32([2]), i32([3])), acc, decay=0.5)
    assert acc[0].tolist() == [3, 3, 1.5, 1.5, 1.5, 3, 3, 3, 3] and torch.equal(acc[0], acc[1])
    assert [t.shape for t in ctx().beam_select(e(0, 3, 50), e(0, 3, dt=torch.float32), 4)] == [(0, 4)] * 3
    parents = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for shape in ((0, 6, 4, 8), (2, 6, 0, 8), (2, 6, 4, 0)):
        assert ctx().beam_reorder(e(*shape), parents).shape == shape
    assert ctx().beam_reorder(e(2, 0, 4, 8), torch.zeros(0, 3, dtype=torch.int32, device="cuda")).shape == (2, 0, 4, 8)
    kept, left = ctx().cache_evict(e(0, 2, 64), e(0, 2, 64), e(2, 0, dt=torch.float32), i32([0, 4]), i32([7, 0]), 5)
    assert torch.all(kept == -1) and left.tolist() == [0, 0]
    v = randn(9, 2, 64, seed=3)
    k0, v0, a0 = k.clone(), v.clone(), acc.clone()
    kept, left = ctx().cache_evict(k, v, acc, i32([]), i32([]), 5)
    assert kept.numel() == 0 and left.numel() == 0
    kept, left = ctx().cache_evict(k, v, acc, i32([1]), i32([8]), 3, k_out=e(0, 2, 64), v_out=e(0, 2, 64), acc_out=e(2, 0, dt=torch.float32))
    assert left.tolist() == [3] and kept.shape == (1, 2, 3)
    assert torch.equal(k, k0) and torch.equal(v, v0) and torch.equal(acc, a0)


# ---- sizes that pass 32 bits ------------------------------------------------------------------


def test_caches_whose_offsets_pass_32_bits():
    """Prefixes, own keys and evicted ones behind 2^31 elements and 2^32 bytes of a cache: the bits of the same call
    where they lie at its begin."""
    import torch
    rows, kv, dim, far = 4_300_000, 4, 128, 4_299_000
    near = 1000
    k, v = (torch.zeros(rows, kv, dim, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    acc = torch.zeros(kv, rows, device="cuda")
    for seed, t in ((1, k), (2, v)):
        t[:near] = randn(near, kv, dim, seed=seed)
        t[far:far + near] = t[:near]
    acc[:, :near] = torch.rand(kv, near, device="cuda")
    acc[:, far:far + near] = acc[:, :near]
    for q_len, n_own in (([1] * 6, 90), ([30] * 6, 90)):
        starts = [sum(q_len[:i]) for i in range(7)]
        q = randn(starts[-1], 8, dim, seed=3, scale=2)
        got, sums = [], []
        for at in (0, far):
            s = vrs.seqs(i32(starts), i32([at + 300 + 100 * i for i in range(6)]), i32([n_own] * 6), max_q=max(q_len), max_k=n_own)
            p = vrs.prefixes(i32([0, 6]), i32([at]), i32([290]), max_rows=starts[-1], max_k=290)
            got.append(ctx().prefix_attention(q, k, v, s, p))
            a = acc.clone()
            ctx().attention_weights(q, k, s, a)
            sums.append(a[:, at:at + near].clone())
            assert torch.equal(a[:, near:far], acc[:, near:far])
        assert got[0].abs().max() > 0 and torch.equal(*got) and torch.equal(*sums)
    kept, left = ctx().cache_evict(k, v, acc, i32([5, far + 5]), i32([900, 900]), 300, first=4, recent=50)
    assert torch.equal(kept[0], kept[1]) and left.tolist() == [300, 300]
    for t in (k, v, acc.t()):
        assert torch.equal(t[:near], t[far:far + near])


def test_beam_states_and_logits_whose_offsets_pass_32_bits():
    import torch
    rows, row = 70, 1 << 20
    state = torch.zeros(2, 32, rows, row, dtype=torch.uint8, device="cuda")             # 4.7 GB
    state[:, ::8] = torch.randint(0, 255, (2, 4, rows, row), dtype=torch.uint8, device="cuda")
    parents = torch.zeros(4, 8, dtype=torch.int32, device="cuda")
    lens = torch.full((32,), 69, dtype=torch.int32, device="cuda")
    ctx().beam_reorder(state, parents, lens=lens)
    for i in range(32):
        assert torch.equal(state[:, i, :69], state[:, i // 8 * 8, :69])
        assert i % 8 == 0 or not state[:, i, 69].any()
    del state
    batch, vocab = 1100, 250000
    x = torch.zeros(batch, 8, vocab, dtype=torch.bfloat16, device="cuda")               # 2.2e9 logits
    x[-1] = logits_of(1, 8, vocab, "bf16", seed=4)[0]
    s = scores_of(batch, 8)
    got = ctx().beam_select(x, s, 8)
    ref = select_ref(x[-1:], s[-1:], 8)
    assert torch.equal(got[1][-1:].cpu(), ref[1]) and torch.equal(got[2][-1:].cpu(), ref[2])
    inside(got[0][-1:].cpu(), ref[0], ref[0].abs() * F * 1.01 + 34 * F * 4)
    assert not got[1][:-1].any() and torch.equal(got[2][:-1].cpu(), torch.arange(8, dtype=torch.int32).expand(batch - 1, 8))

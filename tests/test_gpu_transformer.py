"""Transformer-layer operators (RMS norm, rotary positions, attention) against
their definitions in 64 bits, at the sizes, strides and masks where they can go
wrong, and a run of them together with the convs between.

Tolerances count roundings: a type rounds by at most U[type] of the value
(bfloat16 2^-8, float32 2^-24, e4m3 2^-4), a float32 sum of n terms by n 2^-24
of the sum of their magnitudes."""
import math

import numpy as np
import pytest

from gpu_util import ctx, vrs

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24, "e4m3": 2.0 ** -4}
F = 2.0 ** -24


def tdt(t):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[t]


def randn(*shape, dtype="bf16", seed=0, scale=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(tdt(dtype))


def inside(got, ref, tol):
    """Every element within its tolerance; NaN where the reference has one."""
    import torch
    got = got.double()
    assert got.shape == ref.shape
    same = (got == ref) | (got.isnan() & ref.isnan())
    off = torch.where(same, torch.zeros_like(ref), (got - ref).abs() - tol)
    worst = off.nan_to_num(nan=math.inf).max().item() if off.numel() else 0.0
    assert worst <= 0, (worst, got.flatten()[off.nan_to_num(nan=math.inf).argmax()], ref.flatten()[off.nan_to_num(nan=math.inf).argmax()])


def i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---- RMS norm ------------------------------------------------------------------------


def rms_ref(x, res, w, eps):
    s = x.double() + (res.double() if res is not None else 0)
    return s, s / (s.square().mean(1, keepdim=True) + eps).sqrt() * w.double()


def rms_tol(cols):
    # a thread's squares (<= 32) and a tree of <= 10 + 16 sums, halved by the root; the sum x + res,
    # mean, eps, root, quotient and two products
    return (21 + 8 + 8) * F


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (257, 520), (2, 1001), (33, 1024), (9, 2048), (4, 4095),
                                       (70, 4096), (3, 8200), (2, 16384), (2, 32767), (3, 32768), (4500, 72)])
def test_rms_norm(dtype, rows, cols):
    x, res = randn(rows, cols, dtype=dtype, seed=1, scale=3), randn(rows, cols, dtype=dtype, seed=2)
    w = randn(cols, dtype="f32", seed=3)
    for r in (None, res):
        y, s, scales = ctx().rms_norm(x, w, 1e-5, res=r)
        rs, ry = rms_ref(x, r, w, 1e-5)
        assert scales is None and (s is None) == (r is None)
        inside(y, ry, ry.abs() * (U[dtype] + rms_tol(cols)) * 1.01 + rs.abs() * 2 * F)
        if r is not None:
            inside(s, rs, rs.abs() * U[dtype] * 1.01)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,cols,group", [(1, 16, 16), (5, 128, 32), (37, 640, 128), (3, 640, 64), (20, 4096, 128),
                                             (7, 4096, 4096), (2, 32768, 32768), (11, 16384, 32), (6, 1040, 0), (300, 256, 0)])
def test_rms_norm_e4m3(dtype, rows, cols, group):
    import torch
    x, res = randn(rows, cols, dtype=dtype, seed=1), randn(rows, cols, dtype=dtype, seed=2)
    w = randn(cols, dtype="f32", seed=3)
    x[rows // 2] = 0
    res[rows // 2] = 0            # a row of zeros: scale 1
    step = 0.125 if group == 0 else 0.0
    y, s, scales = ctx().rms_norm(x, w, 1e-6, res=res, e4m3=True, group=group, out_step=step)
    rs, ry = rms_ref(x, res, w, 1e-6)
    inside(s, rs, rs.abs() * U[dtype] * 1.01)
    e = rms_tol(cols)
    if group == 0:
        assert scales is None
        scale = torch.full((rows, cols), step, dtype=torch.float64, device="cuda")
    else:
        amax = ry.abs().view(rows, -1, group).amax(2)
        rscale = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
        inside(scales, rscale, rscale * (e + 4 * F))
        scale = scales.double().repeat_interleave(group, 1)
    # the quotient by the stored scale, clamped: e4m3's relative half step, or half of 2^-9 below 2^-6
    q = (ry / scale).clamp(-448, 448)
    inside(y.view(torch.float8_e4m3fn), q, (q.abs() * U["e4m3"]).clamp(min=2.0 ** -10) + q.abs() * (e + 4 * F) * 1.1 + rs.abs() / scale * 2 * F)


def test_rms_norm_strides_and_in_place():
    """Rows apart from each other, x written over by y, and the residual by the sum; what lies between rows stays."""
    import torch
    for cols, pad in ((256, 8), (250, 3)):
        big = randn(10, cols + pad, seed=4)
        res = randn(10, cols + pad, seed=5)
        w = randn(cols, dtype="f32", seed=6)
        x0, r0 = big.clone(), res.clone()
        rs, ry = rms_ref(x0[:, :cols], r0[:, :cols], w, 1e-6)
        ctx().rms_norm(big[:, :cols], w, 1e-6, res=res[:, :cols], sum=res[:, :cols], y=big[:, :cols])
        inside(big[:, :cols], ry, ry.abs() * (U["bf16"] + rms_tol(cols)) * 1.01 + rs.abs() * 2 * F)
        inside(res[:, :cols], rs, rs.abs() * U["bf16"] * 1.01)
        assert torch.equal(big[:, cols:], x0[:, cols:]) and torch.equal(res[:, cols:], r0[:, cols:])


def test_rms_norm_values_at_the_ends_of_the_range():
    """Squares that leave float32, zeros, infinities and NaN stay inside their row and group."""
    import torch
    x = randn(6, 512, dtype="f32", seed=7)
    x[0] *= 1e30
    x[1] *= 1e-30
    x[2] = 0
    x[3, 5] = math.nan
    x[4, 5] = math.inf
    w = torch.ones(512, device="cuda")
    y, _, _ = ctx().rms_norm(x, w, 1e-37)
    rs, ry = rms_ref(x, None, w, 1e-37)
    inside(y, ry, ry.abs() * (U["f32"] + rms_tol(512)))
    w[5] = math.nan
    x[3:5] = 1.0
    q, _, sc = ctx().rms_norm(x, w, 1e-37, e4m3=True, group=32)
    q = q.view(torch.float8_e4m3fn).float()
    assert q[:, 5].isnan().all() and sc.isfinite().all()
    q[:, 5] = 0
    assert q.isfinite().all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cols,group", [(512, 32), (512, 64), (4096, 128), (256, 256), (4096, 4096), (16384, 128), (16384, 16384)])
def test_rms_norm_e4m3_of_tiny_maxima(dtype, cols, group):
    """Scales that are no normal number, or none at all: quotients by them, and zeros stay zeros."""
    import torch
    x = randn(6, cols, dtype=dtype, seed=8)
    x[:, ::5] = 0
    tiny = [1.0, 3e-36, 2e-37, 1e-38, 1e-40, 3e-42, 2e-44]
    groups = cols // group
    for first in range(0, 7, 1 if groups == 1 else 4):      # one group: its weights are each size in turn
        w = randn(cols, dtype="f32", seed=9).sign()
        for g in range(groups):
            w[g * group:(g + 1) * group] *= tiny[(first + g) % 7]
        y, _, scales = ctx().rms_norm(x, w, 1e-6, e4m3=True, group=group)
        _, ry = rms_ref(x, None, w, 1e-6)
        e = rms_tol(cols)
        # y and the scale are off by half a unit of 2^-149 besides, twice for the maximum's own
        amax = ry.abs().view(6, groups, group).amax(2)
        rscale = amax / 448
        rscale = torch.where(rscale < 2.0 ** -150, torch.ones_like(rscale), rscale)
        inside(scales, rscale, rscale * (e + 4 * F) + 2.0 ** -149)
        scale = scales.double().repeat_interleave(group, 1)
        q = (ry / scale).clamp(-448, 448)
        got = y.view(torch.float8_e4m3fn)
        inside(got, q, (q.abs() * U["e4m3"]).clamp(min=2.0 ** -10) + q.abs() * (e + 4 * F) * 1.1 + 2.0 ** -149 / scale * (1 + U["e4m3"]))
        assert torch.all(got.float()[:, ::5] == 0)


# ---- rotary positions ----------------------------------------------------------------


def rope_ref(x, pos, freq, rot, pairs, scale):
    """x [rows, heads, dim], pos [rows, rot / 2] in 64 bits."""
    import torch
    turn = torch.remainder(pos.double() * freq, 1.0) * (2 * math.pi)
    c, s = turn.cos()[:, None], turn.sin()[:, None]
    y = x.double().clone()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a.double(), b.double()
    ya, yb = scale * (a * c - b * s), scale * (a * s + b * c)
    mag = torch.zeros_like(y)
    m = abs(scale) * (a.abs() + b.abs())
    if pairs:
        y[..., 0:rot:2], y[..., 1:rot:2], mag[..., 0:rot:2], mag[..., 1:rot:2] = ya, yb, m, m
    else:
        y[..., :rot // 2], y[..., rot // 2:rot], mag[..., :rot // 2], mag[..., rot // 2:rot] = ya, yb, m, m
    return y, mag


def rope_inside(got, ref, dtype):
    # the fraction of a turn in float32 (pi 2^-24 of an angle), 4 units for the functions' own error,
    # the scale, two products and a sum: 12 units of |a| + |b|
    y, mag = ref
    inside(got, y, y.abs() * U[dtype] * 1.01 + mag * 12 * F)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("rows,heads,kv,dim,rot", [(1, 1, 1, 2, 2), (3, 2, 1, 64, 64), (130, 5, 2, 80, 40), (7, 4, 4, 72, 72),
                                                   (2050, 8, 2, 128, 128), (9, 3, 1, 50, 22), (5, 1, 1, 1024, 512)])
def test_rope(dtype, pairs, rows, heads, kv, dim, rot):
    import torch
    qkv = randn(rows, heads + kv, dim, dtype=dtype, seed=1)
    q, k = qkv[:, :heads], qkv[:, heads:]
    freq = vrs.rope_freqs(rot // 2).cuda()
    pos = torch.randint(0, 1 << 30, (rows,), device="cuda", dtype=torch.int32)     # far positions
    ref = [rope_ref(x, pos[:, None].expand(rows, rot // 2), freq, rot, pairs, 1.25) for x in (q, k)]
    layout = vrs.ROPE_PAIRS if pairs else vrs.ROPE_HALF
    qo, ko = ctx().rope(q, k, freq, rot_dim=rot, layout=layout, positions=pos, scale=1.25)
    rope_inside(qo, ref[0], dtype)
    rope_inside(ko, ref[1], dtype)
    # in place, the row as the position; one of the two alone
    ref = rope_ref(q, torch.arange(rows, device="cuda")[:, None].expand(rows, rot // 2), freq, rot, pairs, 1.0)
    k0 = k.clone()
    ctx().rope(q, None, freq, rot_dim=rot, layout=layout, q_out=q)
    rope_inside(q, ref, dtype)
    assert torch.equal(k, k0)


@pytest.mark.parametrize("dim,rot,split", [(64, 64, (10, 22)), (80, 60, (0, 14, 16)), (128, 128, (16, 16, 16, 16))])
def test_rope_axes(dim, rot, split):
    import torch
    rows = 77
    k = randn(rows, 3, dim, dtype="f32", seed=1)
    freq = torch.cat([vrs.rope_freqs(n) for n in split if n]).cuda()
    pos = torch.randint(-50, 5000, (len(split), rows + 5), device="cuda", dtype=torch.int32)
    axis = torch.tensor([i for i, n in enumerate(split) for _ in range(n)], device="cuda")
    ref = rope_ref(k, pos[:, :rows].t()[:, axis], freq, rot, True, 1.0)
    _, ko = ctx().rope(None, k, freq, rot_dim=rot, layout=vrs.ROPE_PAIRS, positions=pos, axis_pairs=split)
    rope_inside(ko, ref, "f32")


CASES = {
    # queries of each sequence, earlier keys, first row of its keys in the cache
    "plain": ([3, 0, 130, 1, 0, 64], None, None),
    "cache": ([3, 0, 130, 1, 64], [7, 5, 0, 200, 61], [900, 40, 300, 600, 60]),
    "short": ([5, 9], [-3, -20], [0, 100]),          # fewer keys than queries
    "many": ([1] * 70, list(range(70)), [100 * i for i in range(70)]),
}


def build(case, lead=2, tail=3, max_hint=True):
    """q_start (rows before the first and behind the last sequence belong to none), seqs, lengths."""
    q_len, past, k_at = CASES[case] if isinstance(case, str) else case
    starts = [lead + sum(q_len[:i]) for i in range(len(q_len) + 1)]
    k_len = [max(0, a + b) for a, b in zip(q_len, past)] if past is not None else list(q_len)
    hint = dict(max_q=max(q_len), max_k=max(k_len)) if max_hint else {}
    s = vrs.seqs(i32(starts), None if k_at is None else i32(k_at), None if past is None else i32(k_len), **hint)
    return starts, starts[-1] + tail, k_len, (starts[:-1] if k_at is None else k_at), s


@pytest.mark.parametrize("dtype,dim,rot", [("bf16", 64, 64), ("f32", 40, 24), ("bf16", 36, 22)])
@pytest.mark.parametrize("case", list(CASES))
def test_rope_into_a_cache(dtype, dim, rot, case):
    import torch
    starts, rows, k_len, k_at, s = build(case)
    qkv = randn(rows, 6, dim, dtype=dtype, seed=1)
    q, k, v = qkv[:, :3], qkv[:, 3:5], qkv[:, 4:6]
    freq = vrs.rope_freqs(rot // 2).cuda()
    n_cache = max(rows, max(a + n for a, n in zip(k_at, k_len)) + 4)
    ko, vo = randn(n_cache, 2, dim, dtype=dtype, seed=2), randn(n_cache, 2, dim, dtype=dtype, seed=3)
    qo = randn(rows, 3, dim, dtype=dtype, seed=4)
    rq, rk, rv = qo.double(), ko.double(), vo.double()
    mq, mk = torch.zeros_like(rq), torch.zeros_like(rk)
    for i, n in enumerate(k_len):
        for r in range(starts[i], starts[i + 1]):
            place = n - (starts[i + 1] - starts[i]) + r - starts[i]
            pos = torch.tensor([[float(place)]], device="cuda").expand(1, rot // 2)
            y, m = rope_ref(qkv[r:r + 1, :5], pos, freq, rot, False, 1.0)
            rq[r], mq[r] = y[0, :3], m[0, :3]
            if place >= 0:
                to = k_at[i] + place
                rk[to], mk[to], rv[to] = y[0, 3:], m[0, 3:], v[r].double()
    ctx().rope(q, k, freq, rot_dim=rot, seqs=s, q_out=qo, k_out=ko, v=v, v_out=vo)
    rope_inside(qo, (rq, mq), dtype)
    rope_inside(ko, (rk, mk), dtype)
    assert torch.equal(vo.double(), rv)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rope_into_a_cache_with_heads_outside_rows(dtype):
    """A cache [sequence, head, room, dim], filled and read through strides: the bits of one with rows of heads."""
    import torch
    n, kv, room, dim, q_len, past = 3, 2, 40, 64, [3, 1, 8], [0, 39, 20]
    starts = [0, 3, 4, 12]
    k_len = [a + b for a, b in zip(q_len, past)]
    qkv = randn(12, 4 + 2 * kv, dim, dtype=dtype, seed=1)
    q, k, v = qkv[:, :4], qkv[:, 4:4 + kv], qkv[:, 4 + kv:]
    freq = vrs.rope_freqs(dim // 2).cuda()
    kc, vc = randn(n, kv, room, dim, dtype=dtype, seed=2), randn(n, kv, room, dim, dtype=dtype, seed=3)
    rows = [t.transpose(1, 2).reshape(n * room, kv, dim).clone() for t in (kc, vc)]
    view = [t.as_strided(((n * kv - (kv - 1)) * room, kv, dim), (dim, room * dim, 1)) for t in (kc, vc)]
    outs = []
    for (ko, vo), per in ((rows, room), (view, kv * room)):
        s = vrs.seqs(i32(starts), i32([i * per for i in range(n)]), i32(k_len), max_q=8, max_k=room)
        qo, _ = ctx().rope(q, k, freq, seqs=s, k_out=ko, v=v, v_out=vo)
        outs += [qo, ctx().attention(qo, ko, vo, s)]
    assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
    for a, b in zip((kc, vc), rows):
        assert torch.equal(a, b.view(n, room, kv, dim).transpose(1, 2))


def test_rope_writes_no_row_outside_the_cache():
    """Starts, lengths and rows that do not fit the buffers are cut off."""
    import torch
    q = randn(12, 1, 64, seed=1)
    freq = vrs.rope_freqs(32).cuda()
    ko = torch.full((20, 1, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    guard = ko[4:12]               # the cache that the call knows: rows 4..11 of the buffer
    s = vrs.seqs(i32([0, 4, 8, 500]), i32([6, -3, 2]), i32([4, 4, 4]))
    ctx().rope(q, q, freq, seqs=s, k_out=guard)
    torch.cuda.synchronize()
    assert torch.all(ko[:4] == 7) and torch.all(ko[12:] == 7)
    assert torch.all(ko[10:12].abs().sum((1, 2)) != 7 * 64) and not torch.all(ko[6] == 7)


# ---- attention -----------------------------------------------------------------------


def attention_ref(q, k, v, starts, k_len, k_at, causal, scale, out, dtype):
    """Result and tolerance in 64 bits; `out` holds what rows of no sequence have."""
    import torch
    ref, tol = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64, device=out.device)
    H, G, D = q.shape[1], q.shape[1] // k.shape[1], q.shape[2]
    for i, n in enumerate(k_len):
        a, b = starts[i], starts[i + 1]
        if a == b:
            continue
        Q = q[a:b].double().transpose(0, 1)
        K = k[k_at[i]:k_at[i] + n].double().repeat_interleave(G, 1).transpose(0, 1)
        V = v[k_at[i]:k_at[i] + n].double().repeat_interleave(G, 1).transpose(0, 1)
        seen = torch.ones(b - a, n, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(n, device=q.device)[None] <= (n - (b - a) + torch.arange(b - a, device=q.device))[:, None]
        s = (Q @ K.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        m = s.amax(2, keepdim=True) if n else s.new_full((H, b - a, 1), -math.inf)
        p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
        p = torch.where(seen, p, torch.zeros_like(p))
        Vs = torch.where(V.isfinite(), V, torch.zeros_like(V))
        total = p.sum(2, keepdim=True)
        o = torch.where(total == 0, torch.zeros_like(total), 1 / total) * (p @ Vs)
        # what is not finite reaches the queries that see it: counted apart, since 0 * inf is no 0
        for value in (math.inf, -math.inf, math.nan):
            hit = V.isnan() if value != value else V == value
            if hit.any():
                o = torch.where((seen.double()[None] @ hit.double()) > 0, o + value, o)
        w = p / torch.where(total == 0, torch.ones_like(total), total)
        # a probability rounded by u: u * sum w |v - o| (their sum holds the rounded ones); scores
        # off by e: the same with 2 e; the float32 sums over the keys
        u = 0.0 if dtype == "f32" else U["bf16"]
        big = (Q.abs() @ K.abs().transpose(1, 2) * scale).masked_fill(~seen, 0).amax(2, keepdim=True) if n else 0
        e = (D + 8) * F * big + 8 * F
        of = o.nan_to_num(0, 0, 0)
        if n:
            spread = torch.stack([(w[h][:, :, None] * (Vs[h][None] - of[h][:, None]).abs()).sum(1) for h in range(H)])
            size = w @ Vs.abs()
            t = spread * (u + 2 * e) * 1.02 + size * (2 * n + 70) * F + of.abs() * U[dtype] * 1.01
        else:
            t = torch.zeros_like(o)
        ref[a:b], tol[a:b] = o.transpose(0, 1), t.transpose(0, 1)
    return ref, tol


def check_attention(case, dtype="bf16", heads=4, kv=2, dim=64, causal=True, scale=0.0, hint=True, seed=0, edit=None,
                    views=None, extra=0):
    import torch
    starts, rows, k_len, k_at, s = build(case, max_hint=hint)
    n_k = max(rows, max([a + n for a, n in zip(k_at, k_len)] + [0])) + extra
    if views is None:
        q, k, v = randn(rows, heads, dim, dtype=dtype, seed=seed, scale=2), randn(n_k, kv, dim, dtype=dtype, seed=seed + 1), \
            randn(n_k, kv, dim, dtype=dtype, seed=seed + 2)
        out = torch.full((rows, heads, dim), 5.0, dtype=tdt(dtype), device="cuda")
    else:
        q, k, v, out = views(rows, n_k)
    if edit:
        edit(q, k, v, starts, k_at, k_len)
    ref, tol = attention_ref(q, k, v, starts, k_len, k_at, causal, scale or dim ** -0.5, out, dtype)
    got = ctx().attention(q, k, v, s, causal=causal, scale=scale, out=out)
    torch.cuda.synchronize()
    assert got is out
    inside(got, ref, tol)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (3, 3, 8), (8, 1, 128), (5, 1, 72)])
def test_attention(dtype, causal, case, heads, kv, dim):
    check_attention(case, dtype, heads, kv, dim, causal)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n", [31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 400])
def test_attention_lengths(dtype, n):
    """Whole prompts around the sizes of the tiles."""
    for causal in (True, False):
        check_attention(([n, 1, n - 1], None, None), dtype, 4, 2, 64, causal, seed=n)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q,past", [(1, 0), (1, 1), (1, 31), (1, 32), (1, 127), (1, 5000), (2, 1000), (7, 3000), (16, 777),
                                    (33, 4000), (100, 6000)])
def test_attention_over_a_cache(dtype, q, past):
    """Single tokens and pieces of prompts, keys split among workgroups."""
    for heads, kv, dim in ((8, 1, 128), (4, 4, 64)):
        for causal in (True, False):
            check_attention(([q], [past], [3]), dtype, heads, kv, dim, causal, seed=past)


@pytest.mark.parametrize("dtype,heads,kv,dim,n,q,past,causal", [
    ("bf16", 8, 8, 64, 4, 4200, 0, False), ("bf16", 16, 4, 64, 1, 9000, 0, True), ("bf16", 6, 2, 40, 3, 6000, 2500, True),
    ("bf16", 8, 2, 128, 2, 4500, 0, True), ("bf16", 4, 4, 120, 2, 5000, 0, False), ("f32", 4, 4, 64, 2, 4100, 0, False),
    ("f32", 4, 1, 128, 1, 4700, 0, True), ("f32", 16, 16, 64, 2, 4100, 0, False), ("f32", 16, 16, 128, 1, 4300, 0, True), ("bf16", 16, 16, 64, 1, 2600, 0, True), ("bf16", 8, 8, 128, 90, 300, 40, True),
])
def test_attention_large(dtype, heads, kv, dim, n, q, past, causal):
    """Workgroups of 256 rows, over 64 sequences, many key tiles: rows picked from all of the output.
    Causal: the last values of a sequence are not finite, which only its last queries see."""
    import torch
    rng = np.random.default_rng(q)
    q_len = [int(v) for v in rng.integers(max(1, q - 200), q + 1, n)]
    k_len = [a + past for a in q_len]
    k_at = [int(v) for v in np.cumsum([0] + k_len[:-1])] if past else None
    starts = [int(v) for v in np.cumsum([1] + q_len)]
    rows, n_k = starts[-1] + 2, sum(k_len) + starts[-1] + 2
    s = vrs.seqs(i32(starts), i32(k_at) if past else None, i32(k_len) if past else None, max_q=max(q_len), max_k=max(k_len))
    qt, k, v = (randn(rows, heads, dim, dtype=dtype, seed=1, scale=2), randn(n_k, kv, dim, dtype=dtype, seed=2),
                randn(n_k, kv, dim, dtype=dtype, seed=3))
    at = k_at if past else starts[:-1]
    if causal:
        for a, m in zip(at, k_len):
            v[a + m - 1, 0, 3], v[a + m - 2, kv - 1, 5] = math.nan, -math.inf
    out = torch.full_like(qt, 5.0)
    ctx().attention(qt, k, v, s, causal=causal, out=out)
    assert torch.all(out[:1] == 5) and torch.all(out[-2:] == 5)
    for i in sorted({0, n // 2, n - 1}):
        for j in sorted({0, 1, 31, 32, 127, 128, 255, 256, q_len[i] // 2, q_len[i] - 1} & set(range(q_len[i]))):
            row, keys = starts[i] + j, k_len[i] - q_len[i] + j + 1 if causal else k_len[i]
            ref, tol = attention_ref(qt[row:row + 1], k, v, [0, 1], [keys], [at[i]], False, dim ** -0.5, out[row:row + 1], dtype)
            inside(out[row:row + 1], ref, tol)


def test_attention_over_its_queries():
    """out may be q."""
    import torch
    for case in ("cache", ([1], [3000], [0]), ([200], [1500], [0])):
        starts, rows, k_len, k_at, s = build(case)
        n_k = max(rows, max(a + n for a, n in zip(k_at, k_len)))
        q, k, v = randn(rows, 4, 64, seed=1), randn(n_k, 2, 64, seed=2), randn(n_k, 2, 64, seed=3)
        want = ctx().attention(q, k, v, s, out=q.clone())
        assert torch.equal(ctx().attention(q, k, v, s, out=q), want)


def test_nothing_to_do():
    """No rows, no sequences, no keys."""
    import torch
    w = torch.ones(64, device="cuda")
    y, s_, _ = ctx().rms_norm(randn(0, 64), w, res=randn(0, 64))
    assert y.shape == s_.shape == (0, 64)
    freq = vrs.rope_freqs(32).cuda()
    assert ctx().rope(randn(0, 2, 64), randn(0, 1, 64), freq)[0].shape == (0, 2, 64)
    q, k = randn(5, 2, 64, seed=1), randn(4, 1, 64, seed=2)
    for s in (vrs.seqs(i32([0])), vrs.seqs(i32([0, 0, 0])), vrs.seqs(i32([5, 5]), i32([0]), i32([3]))):
        out = ctx().attention(q, k, k, s, out=torch.full_like(q, 5.0))
        assert torch.all(out == 5)
    for max_q in (0, 5, 1000):
        s = vrs.seqs(i32([1, 4]), i32([0]), i32([0]), max_q=max_q, max_k=0)
        out = ctx().attention(q, k[:0], k[:0], s, out=torch.full_like(q, 5.0))
        assert torch.all(out[1:4] == 0) and torch.all(out[0] == 5) and torch.all(out[4] == 5)


def test_attention_given_workspace():
    """A workspace of the size asked for, full of NaN; one byte less is refused."""
    import ctypes as C
    import torch
    starts, rows, k_len, k_at, s = build(([1], [5000], [0]))
    q, k, v = randn(rows, 4, 64, seed=1), randn(5001, 1, 64, seed=2), randn(5001, 1, 64, seed=3)
    want = ctx().attention(q, k, v, s, out=torch.zeros_like(q))
    d = vrs.AttentionDesc(rows, 5001, 4, 1, 64, vrs.BF16, 1, 0.0, 256, 64, 64, 64, 64, 64, 256, 64)
    need = vrs.lib().vrs_attention_workspace_size(C.byref(d), s.address)
    assert need > 0
    ws = torch.full((need // 4,), math.nan, device="cuda").view(torch.uint8)
    assert torch.equal(ctx().attention(q, k, v, s, out=torch.zeros_like(q), workspace=ws), want)
    with pytest.raises(vrs.VrsError) as e:
        ctx().attention(q, k, v, s, workspace=ws[:-16])
    assert e.value.code == -1


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (8, 2, 128)])
def test_attention_pieces_and_tokens_in_one_call(dtype, heads, kv, dim):
    """A prompt, pieces and single tokens over long and short caches: workgroups most of whose waves have no row."""
    case = ([1, 300, 1, 70, 1, 5, 1], [2500, 0, 900, 1500, 0, 40, 130], [0, 2600, 3000, 4000, 5700, 5800, 5900])
    for causal in (True, False):
        check_attention(case, dtype, heads, kv, dim, causal)


def test_attention_hints_choose_kernels_only():
    """Unknown, too small and too large hints: right results of every kernel."""
    import torch
    for case in ("cache", ([1, 1, 1], [700, 3, 900], [0, 800, 1000]), ([300], [2000], [0])):
        starts, rows, k_len, k_at, s = build(case)
        n_k = max(rows, max(a + n for a, n in zip(k_at, k_len)))
        q, k, v = randn(rows, 4, 64, seed=1, scale=2), randn(n_k, 2, 64, seed=2), randn(n_k, 2, 64, seed=3)
        out = torch.zeros(rows, 4, 64, dtype=torch.bfloat16, device="cuda")
        ref, tol = attention_ref(q, k, v, starts, k_len, k_at, True, 0.125, out, "bf16")
        for max_q, max_k in ((0, 0), (1, 1), (1, 0), (5, 4000), (1 << 30, 1 << 30), (64, 1)):
            s.max_q, s.max_k = max_q, max_k
            inside(ctx().attention(q, k, v, s, out=out.clone()), ref, tol)


def test_attention_scale_and_large_scores():
    for dtype in ("bf16", "f32"):
        check_attention("cache", dtype, scale=3.0)          # near one-hot rows
        check_attention("cache", dtype, scale=1e-4)
        check_attention(([70], None, None), dtype, scale=1e-30)


LARGE = [(1, 60, 4, 2, 64), (1, 5000, 8, 1, 128), (3, 900, 4, 2, 64), (130, 0, 4, 2, 64), (100, 6000, 8, 1, 128), (2100, 0, 32, 32, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("base,step", [(2.0 ** 20, 1.0), (2.0 ** 20, 0.25), (-2.0 ** 20, 1.0), (-2.0 ** 31, 2.0 ** 12), (2.0 ** 40, 2.0 ** 30), (-2.0 ** 40, 2.0 ** 30),
                                       (-2.0 ** 100, 2.0 ** 90), (2.0 ** 100, 2.0 ** 90), (-2.0 ** 29, 2.0 ** 6), (0.0, 2.0 ** 60), (0.0, 2.0 ** 28), (0.0, 2.0 ** 110)])
@pytest.mark.parametrize("q_len,past,heads,kv,dim", LARGE)
def test_attention_scores_far_from_zero(dtype, base, step, q_len, past, heads, kv, dim):
    """Scores that float32 holds exactly, all far below or above zero or growing from one to the other:
    base + step * level, the level a key's own."""
    import torch
    n = q_len + past
    causal = q_len < 1000
    g = torch.Generator(device="cuda").manual_seed(q_len)
    level = torch.randint(0, 5 if step > 0.5 else 60, (n,), generator=g, device="cuda")
    if base == 0:
        level = torch.arange(n, device="cuda") * 5 // n - 2       # rising
    q = torch.zeros(q_len, heads, dim, dtype=tdt(dtype), device="cuda")
    k = torch.zeros(n, kv, dim, dtype=tdt(dtype), device="cuda")
    half = 2.0 ** (math.log2(abs(base)) // 2) if base else 0.0
    q[..., 0], q[..., dim - 1] = half, step ** 0.5 if step > 1 else 1.0
    k[..., 0], k[..., dim - 1] = (base / half if base else 0.0), level[:, None] * (step / q[0, 0, dim - 1].item())
    v = randn(n, kv, dim, dtype=dtype, seed=3)
    s = base + step * level.double()
    assert torch.equal((q[0, 0].double() @ k[:, 0].double().t()), s) and torch.equal(s.float().double(), s)
    seqs = vrs.seqs(i32([0, q_len]), i32([0]), i32([n]), max_q=q_len, max_k=n)
    got = ctx().attention(q, k, v, seqs, causal=causal, scale=1.0)
    seen = torch.ones(q_len, n, dtype=torch.bool, device="cuda")
    if causal:
        seen = seen.tril(past)
    s = s[None].masked_fill(~seen, -math.inf)
    w = torch.softmax(s, 1)
    vd = v.double().repeat_interleave(heads // kv, 1)
    ref = (w @ vd.view(n, -1)).view(q_len, heads, dim)
    size = (w @ vd.abs().view(n, -1)).view(q_len, heads, dim)
    # as in attention_ref, the scores exact: exponents under 2^5 of half a unit, and a function off by one
    u = 0.0 if dtype == "f32" else U["bf16"]
    inside(got, ref, (size + ref.abs()) * (u + 64 * F) * 1.02 + size * (2 * n + 70) * F + ref.abs() * U[dtype] * 1.01)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q_len,past,heads,kv,dim", LARGE[:5])
def test_attention_scores_all_minus_infinity(dtype, q_len, past, heads, kv, dim):
    """A query all of whose keys score -inf has no weights: NaN, not the 0 of one that sees no key; such keys
    weigh nothing beside others."""
    import torch
    for lost in (5, past + 5, q_len + past):              # keys from the first on that score -inf
        lost = min(lost, q_len + past)
        n_k = past + max(q_len - 3, 1)                    # a prompt's first queries see none
        lost = min(lost, n_k)
        starts, k_at, k_len = [0, q_len], [2], [n_k]
        q, k, v = randn(q_len, heads, dim, dtype=dtype, seed=1), randn(n_k + 4, kv, dim, dtype=dtype, seed=2), \
            randn(n_k + 4, kv, dim, dtype=dtype, seed=3)
        q[..., 1] = 1.0
        out = torch.zeros_like(q)
        seqs = vrs.seqs(i32(starts), i32(k_at), i32(k_len), max_q=q_len, max_k=n_k)
        ref, tol = attention_ref(q, k, v, starts, [n_k - lost], [2 + lost], True, dim ** -0.5, out, dtype)
        sees = n_k - q_len + torch.arange(q_len, device="cuda") + 1      # keys of each query
        ref[(sees > 0) & (sees <= lost)] = math.nan
        k[2:2 + lost, :, 1] = -math.inf
        inside(ctx().attention(q, k, v, seqs, out=out), ref, tol)


def test_attention_strided():
    """Queries, keys and values of one product; heads outermost; a repeated head."""
    import torch
    def fused(rows, n_k):
        t = randn(max(rows, n_k), 12 * 64 + 16, seed=1)
        cut = lambda a, n, r: t[:r, a * 64:(a + n) * 64].view(r, n, 64)   # noqa: E731
        return cut(0, 8, rows), cut(8, 2, n_k), cut(10, 2, n_k), torch.full((rows, 8, 80), 5.0, dtype=torch.bfloat16, device="cuda")[..., :64]
    def outer(rows, n_k):
        f = lambda n, r, sd: randn(n, r, 64, seed=sd).transpose(0, 1)   # noqa: E731
        return f(8, rows, 1), f(2, n_k, 2), f(2, n_k, 3), torch.full((8, rows, 64), 5.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    def repeated(rows, n_k):
        return (randn(rows, 8, 64, seed=1), randn(n_k, 1, 64, seed=2).expand(n_k, 2, 64), randn(n_k, 1, 64, seed=3).expand(n_k, 2, 64),
                torch.full((rows, 8, 64), 5.0, dtype=torch.bfloat16, device="cuda"))
    for views in (fused, outer, repeated):
        for case in ("plain", "many"):
            check_attention(case, heads=8, kv=2, views=views)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("case", ["plain", "cache", "many", ([5], [300], [1]), ([150], [1300], [1])])
def test_attention_not_finite_in_masked_places(dtype, case):
    """Infinities and NaN at keys that a query does not see leave it alone, and reach those that do."""
    import torch
    def behind(q, k, v, starts, k_at, k_len):      # everything that is no sequence's key
        used = torch.zeros(k.shape[0], dtype=torch.bool, device="cuda")
        for a, n in zip(k_at, k_len):
            used[a:a + n] = True
        k[~used], v[~used] = math.nan, math.inf
    for causal in (True, False):
        check_attention(case, dtype, 4, 2, 64, causal, edit=behind, extra=70)
    def future(q, k, v, starts, k_at, k_len):      # the last keys of each sequence: values not finite
        for i, (a, n) in enumerate(zip(k_at, k_len)):
            if n > 3:
                v[a + n - 1, 0, 3], v[a + n - 1, 0, 40] = math.nan, math.inf
                v[a + n - 2, 1, 5], v[a + n - 3, 1, 5] = math.inf, -math.inf
                v[a + n // 2, 1, 63] = -math.inf
    check_attention(case, dtype, 4, 2, 64, True, edit=future)
    def lowest(q, k, v, starts, k_at, k_len):      # keys whose scores are the type's lowest, finite
        for a, n in zip(k_at, k_len):
            v[a:a + n] = v[a:a + n].abs()
    check_attention(case, dtype, 4, 2, 64, True, edit=lowest)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [8, 24, 40, 56, 72, 80, 96, 120])
def test_attention_narrow_heads_after_full_ones(dtype, dim):
    """What earlier kernels left in LDS does not reach heads narrower than their tile."""
    import torch
    for case, big in ((([200, 33], None, None), ([9000, 9000], None, None)), (([1, 2], [700, 40], [0, 800]), ([1] * 300, [64] * 300, list(range(300))))):
        starts, rows, k_len, k_at, s = build(big)
        n_k = max(rows, max(a + n for a, n in zip(k_at, k_len)))
        nan = torch.full((n_k, 4, 128), math.nan, dtype=tdt(dtype), device="cuda")
        for _ in range(2):         # prompts: a workgroup to each CU at least, and in it 96 KB, the most that these use
            assert ctx().attention(torch.ones_like(nan[:rows]), nan, nan, s, causal=False)[starts[0]:starts[-1]].isnan().all()
        for causal in (True, False):
            check_attention(case, dtype, 4, 2, dim, causal)


def test_attention_nan_keys():
    """A NaN key: NaN for the queries that see it, nothing for the others."""
    import torch
    starts, rows, k_len, k_at, s = build(([90], None, None))
    q, k, v = randn(rows, 2, 64, seed=1), randn(rows, 2, 64, seed=2), randn(rows, 2, 64, seed=3)
    clean = ctx().attention(q, k, v, s).clone()
    k[k_at[0] + 50, 1, 7] = math.nan
    got = ctx().attention(q, k, v, s)
    a = starts[0]
    assert torch.equal(got[a:a + 90, 0], clean[a:a + 90, 0]) and torch.equal(got[a:a + 50, 1], clean[a:a + 50, 1])
    assert got[a + 50:a + 90, 1].isnan().all()


def test_attention_keys_outside_the_buffer_are_cut_off():
    """Lengths and starts past k_rows: the keys inside count, nothing else is read or written."""
    import torch
    q, buf = randn(6, 2, 64, seed=1), randn(40, 2, 64, seed=2)
    k = buf[:20]
    buf[20:] = math.nan
    out = torch.full((10, 2, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    s = vrs.seqs(i32([0, 2, 4, 900]), i32([10, 50, -1]), i32([1000, 5, 5]), max_q=2, max_k=1000)
    ctx().attention(q, k, k, s, causal=False, out=out[:6])
    ref, tol = attention_ref(q[:2], k, k, [0, 2], [10], [10], False, 0.125, out[:2], "bf16")
    inside(out[:2], ref, tol)
    assert torch.all(out[2:6] == 0) and torch.all(out[6:] == 5)


def test_attention_far_into_a_large_cache():
    """Keys past 2^32 bytes and 2^31 elements of one buffer."""
    import torch
    rows, dim = (1 << 31) // (2 * 128) + 5000, 128
    k = torch.empty(rows, 2, dim, dtype=torch.bfloat16, device="cuda")
    at = rows - 3000
    k[at:] = randn(3000, 2, dim, seed=1)
    q = randn(5, 4, dim, seed=2)
    for n_q, n_k in ((1, 2500), (5, 2900)):
        s = vrs.seqs(i32([0, n_q]), i32([at + 7]), i32([n_k]), max_q=n_q, max_k=n_k)
        out = ctx().attention(q[:n_q], k, k, s)
        ref, tol = attention_ref(q[:n_q], k[at:], k[at:], [0, n_q], [n_k], [7], True, dim ** -0.5, out, "bf16")
        inside(out, ref, tol)
    freq = vrs.rope_freqs(64).cuda()
    s = vrs.seqs(i32([0, 5]), i32([at]), i32([2000]), max_q=5, max_k=2000)
    kq = randn(5, 2, dim, seed=3)
    ctx().rope(None, kq, freq, seqs=s, k_out=k)
    y, m = rope_ref(kq, torch.arange(1995, 2000, device="cuda")[:, None].expand(5, 64), freq, dim, False, 1.0)
    rope_inside(k[at + 1995:at + 2000], (y, m), "bf16")


def test_attention_is_the_same_every_time():
    """Fixed order of every sum, also where the keys are split."""
    import torch
    for case in (([1], [5000], [0]), ([200], [3000], [0]), "cache"):
        starts, rows, k_len, k_at, s = build(case)
        n_k = max(rows, max(a + n for a, n in zip(k_at, k_len)))
        q, k, v = randn(rows, 4, 64, seed=1), randn(n_k, 1, 64, seed=2), randn(n_k, 1, 64, seed=3)
        first = ctx().attention(q, k, v, s, out=torch.zeros_like(q)).clone()
        for _ in range(5):
            assert torch.equal(ctx().attention(q, k, v, s, out=torch.zeros_like(q)), first)


# ---- streams, graphs, a run of all -----------------------------------------------------


def test_layers_in_a_graph_follow_the_device_lengths():
    """One captured step of single tokens: replayed while the lengths on the device grow."""
    import torch
    n, H, KV, D, cap = 3, 8, 2, 64, 900
    x = randn(n, H * D, seed=1)
    w = randn(H * D, dtype="f32", seed=2)
    qkv = randn(n, H + 2 * KV, D, seed=3)
    kc, vc = randn(n * cap, KV, D, seed=4), randn(n * cap, KV, D, seed=5)
    freq = vrs.rope_freqs(D // 2).cuda()
    lens = i32([5, 300, 640])
    s = vrs.seqs(i32([0, 1, 2, 3]), i32([0, cap, 2 * cap]), lens, max_q=1, max_k=cap)

    def step():
        y, _, _ = ctx().rms_norm(x, w)
        q, _ = ctx().rope(qkv[:, :H], qkv[:, H:H + KV], freq, seqs=s, k_out=kc, v=qkv[:, H + KV:], v_out=vc)
        return y, ctx().attention(q, kc, vc, s)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gy, go = step()
    for i in range(4):
        lens += 1 + 40 * i
        qkv.copy_(randn(n, H + 2 * KV, D, seed=10 + i))
        kept = kc.clone(), vc.clone()
        ey, eo = step()
        want = ey.clone(), eo.clone(), kc.clone(), vc.clone()
        kc.copy_(kept[0])
        vc.copy_(kept[1])
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip((gy, go, kc, vc), want):
            assert torch.equal(a, b), i


def test_layers_on_two_streams():
    """Calls that overlap, each with its own workspace; an explicit stream."""
    import torch
    s = vrs.seqs(i32([0, 1]), i32([0]), i32([4000]), max_q=1, max_k=4000)
    sets = [(randn(1, 8, 128, seed=i), randn(4000, 1, 128, seed=20 + i), randn(4000, 1, 128, seed=40 + i)) for i in range(4)]
    want = [ctx().attention(*t, s).clone() for t in sets]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [ctx().attention(*t, s, stream=streams[i % 2].cuda_stream) for i, t in enumerate(sets * 5)]
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


def test_a_layer_of_all_operators():
    """A pre-norm attention layer over packed images: norm (e4m3 on the step that the fp8 conv reads), a 1x1
    conv as the product for q, k and v, rotary positions on two axes, attention, a 1x1 conv back, norm
    with the residual.  Each step against its own definition on what it was given."""
    import torch
    H, D, sizes = 4, 64, [(14, 14), (9, 17), (1, 3)]
    C = H * D
    lens = [a * b for a, b in sizes]
    rows = sum(lens)
    starts = [sum(lens[:i]) for i in range(len(lens) + 1)]
    s = vrs.seqs(i32(starts), max_q=max(lens), max_k=max(lens))
    pos = i32([[r for a, b in sizes for r in range(a) for _ in range(b)], [c for a, b in sizes for _ in range(a) for c in range(b)]])
    x, w1 = randn(rows, C, seed=1), 1 + 0.1 * randn(C, dtype="f32", seed=2)
    step = 2.0 ** -6
    y8, _, _ = ctx().rms_norm(x, w1, e4m3=True, out_step=step)
    rs, ry = rms_ref(x, None, w1, 1e-6)
    q8 = (ry / step).clamp(-448, 448)
    inside(y8.view(torch.float8_e4m3fn), q8, (q8.abs() * U["e4m3"]).clamp(min=2.0 ** -10) + q8.abs() * 60 * F)

    rng = np.random.default_rng(0)
    wq = (rng.standard_normal((3 * C, C, 1, 1)) * C ** -0.5).astype(np.float32)
    packed, sc = vrs.pack_conv_weight_fp8(wq)
    qkv = torch.empty(1, 1, rows, 3 * C, dtype=torch.bfloat16, device="cuda")
    ctx().conv2d(vrs.nhwc(y8.view(1, 1, rows, C)), torch.from_numpy(packed).cuda(), torch.from_numpy(sc * step).cuda(),
                 torch.zeros(3 * C, device="cuda"), vrs.nhwc(qkv), 1, act=vrs.ACT_NONE, dtype=vrs.FP8, in_scale=step, x_e4m3=True)
    w_deq = torch.from_numpy(packed).cuda().view(torch.float8_e4m3fn).double().view(3 * C, C) * torch.from_numpy(sc).cuda().double()[:, None]
    x_deq = y8.view(torch.float8_e4m3fn).double() * step
    prod = x_deq @ w_deq.t()
    inside(qkv.view(rows, 3 * C), prod, prod.abs() * U["bf16"] * 1.01 + (x_deq.abs() @ w_deq.abs().t()) * (C + 8) * F)

    t = qkv.view(rows, 3 * H, D)
    q, k, v = t[:, :H], t[:, H:2 * H], t[:, 2 * H:]
    freq = torch.cat([vrs.rope_freqs(D // 4, 100.0)] * 2).cuda()
    axis = torch.tensor([0] * (D // 4) + [1] * (D // 4), device="cuda")
    want = [rope_ref(a, pos.t()[:, axis], freq, D, False, 1.0) for a in (q, k)]
    qo, ko = ctx().rope(q, k, freq, seqs=s, positions=pos, axis_pairs=(D // 4, D // 4))
    rope_inside(qo, want[0], "bf16")
    rope_inside(ko, want[1], "bf16")

    o = ctx().attention(qo, ko, v, s, causal=False)
    inside(o, *attention_ref(qo, ko, v, starts, lens, starts[:-1], False, D ** -0.5, o, "bf16"))

    wo = (rng.standard_normal((C, C, 1, 1)) * C ** -0.5).astype(np.float32)
    z = torch.empty(1, 1, rows, C, dtype=torch.bfloat16, device="cuda")
    wo_p = torch.from_numpy(vrs.pack_conv_weight(wo)).cuda()
    ctx().conv2d(vrs.nhwc(o.view(1, 1, rows, C)), wo_p, torch.ones(C, device="cuda"), torch.zeros(C, device="cuda"),
                 vrs.nhwc(z), 1, act=vrs.ACT_NONE)
    wo_d = wo_p.view(torch.bfloat16).double().view(C, C)
    prod = o.view(rows, C).double() @ wo_d.t()
    inside(z.view(rows, C), prod, prod.abs() * U["bf16"] * 1.01 + (o.view(rows, C).double().abs() @ wo_d.abs().t()) * (C + 8) * F)

    y, h, _ = ctx().rms_norm(z.view(rows, C), w1, res=x)
    rs, ry = rms_ref(z.view(rows, C), x, w1, 1e-6)
    inside(h, rs, rs.abs() * U["bf16"] * 1.01)
    inside(y, ry, ry.abs() * (U["bf16"] + rms_tol(C)) * 1.01 + rs.abs() * 2 * F)

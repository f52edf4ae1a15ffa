"""CPU-side checks of the transformer-layer operators: what they refuse, before
any HIP call, and the host's frequencies of rotary positions."""
import ctypes as C
import math

import pytest

from gpu_util import vrs

FAKE = 1 << 20        # stands for a device address: no refused call follows it


@pytest.fixture()
def ctx():
    return C.cast(C.create_string_buffer(4096), C.c_void_p)   # never read: every call here is refused or empty


def _code(rc):
    return rc, vrs.lib().vrs_last_error().decode()


# ---- rms norm -------------------------------------------------------------------


def rms(ctx, x=FAKE, res=None, w=FAKE, s=None, y=2 * FAKE, scales=None, **kw):
    d = vrs.RmsDesc(rows=4, cols=64, dtype=vrs.BF16, y_dtype=vrs.BF16, eps=1e-6, x_ld=64, res_ld=64, sum_ld=64, y_ld=64)
    for k, v in kw.items():
        setattr(d, k, v)
    return _code(vrs.lib().vrs_rms_norm(ctx, C.byref(d), x, res, w, s, y, scales, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(x=None)), (-1, dict(w=None)), (-1, dict(y=None)),
    (-3, dict(dtype=7)), (-3, dict(y_dtype=vrs.F32)), (-2, dict(rows=-1)), (-2, dict(cols=0)),
    (-3, dict(cols=32769, x_ld=40000, y_ld=40000)), (-1, dict(eps=0.0)), (-1, dict(eps=-1.0)), (-1, dict(eps=math.nan)),
    (-2, dict(y_ld=63)), (-2, dict(x_ld=-64)), (-2, dict(x_ld=1 << 41)), (-2, dict(s=3 * FAKE, sum_ld=8)), (-2, dict(x=FAKE + 1)),
    (-1, dict(s=2 * FAKE)), (-2, dict(y=FAKE, y_ld=128)), (-1, dict(group=32)),
    # e4m3
    (-1, dict(y_dtype=vrs.FP8)), (-1, dict(y_dtype=vrs.FP8, out_step=0.3)), (-1, dict(y_dtype=vrs.FP8, out_step=-1.0)),
    (-3, dict(y_dtype=vrs.FP8, group=16, scales=FAKE)), (-2, dict(y_dtype=vrs.FP8, group=128, scales=FAKE)),
    (-1, dict(y_dtype=vrs.FP8, group=32)), (-2, dict(y_dtype=vrs.FP8, group=32, scales=FAKE + 2)),
    (-1, dict(y_dtype=vrs.FP8, out_step=1.0, y=FAKE)), (-2, dict(y_dtype=vrs.FP8, out_step=1.0, x=FAKE + 2)),
    (-2, dict(y_dtype=vrs.FP8, out_step=1.0, cols=24, x_ld=24)), (-2, dict(y_dtype=vrs.FP8, out_step=1.0, y_ld=72)),
])
def test_rms_norm_refuses(ctx, code, kw):
    rc, msg = rms(ctx, **kw)
    assert rc == code and "vrs_rms_norm" in msg, (rc, msg)


def test_rms_norm_of_no_rows_is_nothing(ctx):
    assert rms(ctx, rows=0)[0] == 0
    assert rms(ctx, rows=0, x=None, y=None)[0] == 0          # an empty tensor's address
    assert vrs.lib().vrs_rms_norm(None, None, None, None, None, None, None, None, None) == -1


# ---- rotary positions -------------------------------------------------------------


def rope(ctx, freq=FAKE, pos=None, q=FAKE, k=2 * FAKE, v=None, qo=3 * FAKE, ko=4 * FAKE, vo=None, seqs=None, **kw):
    d = vrs.RopeDesc(rows=4, k_out_rows=4, heads=2, kv_heads=1, head_dim=64, rot=64, layout=0, dtype=vrs.BF16, axes=1,
                     axis_pairs=(C.c_int32 * 4)(32, 0, 0, 0), scale=1.0, pos_ld=4, q_ld=128, q_hd=64, k_ld=64, k_hd=64,
                     v_ld=64, v_hd=64, qo_ld=128, qo_hd=64, ko_ld=64, ko_hd=64, vo_ld=64, vo_hd=64)
    for key, val in kw.items():
        setattr(d, key, (C.c_int32 * 4)(*val) if key == "axis_pairs" else val)
    s = C.byref(seqs) if seqs is not None else None
    return _code(vrs.lib().vrs_rope(ctx, C.byref(d), s, freq, pos, q, k, v, qo, ko, vo, None))


MOVED = vrs.Seqs(FAKE, FAKE, FAKE, 1, 0, 0)


@pytest.mark.parametrize("code,kw", [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(qo=None)), (-1, dict(ko=None)), (-1, dict(freq=None)),
    (-2, dict(freq=FAKE + 4)), (-3, dict(dtype=2)), (-2, dict(rot=63)), (-2, dict(rot=66)), (-2, dict(rot=0)),
    (-2, dict(heads=0, kv_heads=0)), (-2, dict(heads=-1)), (-2, dict(rows=-1)), (-1, dict(layout=2)),
    (-1, dict(scale=math.inf)), (-1, dict(axes=0)), (-1, dict(axes=5, pos=FAKE)), (-1, dict(axes=2)),
    (-2, dict(axes=2, pos=FAKE, axis_pairs=(16, 15, 0, 0))), (-2, dict(axes=2, pos=FAKE, axis_pairs=(33, -1, 0, 0))),
    (-2, dict(pos=FAKE, pos_ld=3)), (-2, dict(pos=FAKE + 1)), (-2, dict(k_out_rows=3)), (-2, dict(q_ld=-1)),
    (-2, dict(qo_ld=32)), (-2, dict(qo_hd=0)), (-2, dict(ko_ld=0)), (-2, dict(qo=FAKE, q_ld=256)),
    (-2, dict(qo_ld=64)), (-2, dict(qo_hd=32)), (-2, dict(q_hd=1 << 41)),
    (-2, dict(ko=2 * FAKE, seqs=MOVED)), (-1, dict(v=5 * FAKE)), (-1, dict(v=5 * FAKE, vo=5 * FAKE)),
    (-1, dict(kv_heads=0, v=5 * FAKE, vo=6 * FAKE)), (-1, dict(seqs=vrs.Seqs(None, None, None, 1, 0, 0))),
    (-2, dict(seqs=vrs.Seqs(FAKE, None, None, -1, 0, 0))), (-2, dict(head_dim=5000)), (-2, dict(head_dim=1024, rot=514)),
])
def test_rope_refuses(ctx, code, kw):
    rc, msg = rope(ctx, **kw)
    assert rc == code and "vrs_rope" in msg, (rc, msg)


@pytest.mark.parametrize("kw", [dict(ko_ld=32), dict(ko_hd=32), dict(v=5 * FAKE, vo=6 * FAKE, vo_ld=63), dict(v=5 * FAKE, vo=6 * FAKE, vo_hd=0)])
def test_rope_refuses_caches_that_fold(ctx, kw):
    """Rows of one head, or heads of one row, on each other, wherever k_start puts them."""
    rc, msg = rope(ctx, seqs=MOVED, **dict(dict(kv_heads=2, k_ld=128, ko_ld=64, ko_hd=256, vo_ld=64, vo_hd=256, k_out_rows=20), **kw))
    assert rc == -2 and "fold" in msg, (rc, msg)


def test_rope_of_no_rows_is_nothing(ctx):
    assert rope(ctx, rows=0)[0] == 0
    assert rope(ctx, rows=0, q=None, k=None, qo=None, ko=None)[0] == 0
    assert rope(ctx, seqs=vrs.Seqs(FAKE, FAKE, FAKE, 0, 0, 0))[0] == 0


def test_rope_frequencies():
    import torch
    pairs, base = 40, 10000.0
    plain = torch.tensor([base ** (-i / pairs) / (2 * math.pi) for i in range(pairs)], dtype=torch.float64)
    assert torch.allclose(vrs.rope_freqs(pairs, base), plain, rtol=1e-14, atol=0)
    assert torch.allclose(vrs.rope_freqs(pairs, base, vrs.ROPE_LINEAR, 4.0), plain / 4, rtol=1e-14, atol=0)
    f = vrs.rope_freqs(pairs, base, vrs.ROPE_BY_TURNS, 8.0, 1.0, 4.0, 4096)
    turns = plain * 4096
    assert torch.allclose(f[turns >= 4], plain[turns >= 4], rtol=1e-14, atol=0)
    assert torch.allclose(f[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
    keep = (turns - 1) / 3
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and torch.allclose(f[mid], (plain * keep + plain / 8 * (1 - keep))[mid], rtol=1e-13, atol=0)
    f = vrs.rope_freqs(pairs, base, vrs.ROPE_BY_INDEX, 8.0, 1.0, 32.0, 4096)
    index = [pairs * math.log(4096 / (t * 2 * math.pi)) / math.log(base) for t in (32.0, 1.0)]
    lo, hi = math.floor(index[0]), math.ceil(index[1])
    share = f / plain
    assert torch.allclose(share[:lo + 1], torch.ones(lo + 1, dtype=torch.float64), rtol=1e-13, atol=0)
    assert torch.allclose(share[hi:], torch.full((pairs - hi,), 0.125, dtype=torch.float64), rtol=1e-13, atol=0)
    assert torch.all(share[lo:hi + 1].diff() < 0)


@pytest.mark.parametrize("pairs,base,orig,lo,hi", [
    (64, 10000.0, 65536, 40, 65), (64, 10000.0, 131072, 45, 70), (32, 10000.0, 65536, 20, 33), (8, 100.0, 32768, 8, 15),
    (8, 100.0, 131072, 11, 15), (64, 10000.0, 100, 0, 20)])
def test_rope_frequencies_whose_ramp_passes_the_last_pair(pairs, base, orig, lo, hi):
    """By index: the ramp ends at the index of `low` turns, which may lie past the last pair (up to 2 pairs - 1) and
    whose first may lie before the first pair."""
    import torch
    at = [pairs * math.log(orig / (t * 2 * math.pi)) / math.log(base) for t in (32.0, 1.0)]
    assert lo == max(math.floor(at[0]), 0) and hi == min(math.ceil(at[1]), 2 * pairs - 1)
    f = vrs.rope_freqs(pairs, base, vrs.ROPE_BY_INDEX, 8.0, 1.0, 32.0, orig)
    for i in range(pairs):
        plain = base ** (-i / pairs) / (2 * math.pi)
        keep = 1 - min(max((i - lo) / (hi - lo), 0.0), 1.0)
        assert math.isclose(f[i].item(), plain * keep + plain / 8 * (1 - keep), rel_tol=1e-12), i


@pytest.mark.parametrize("args", [
    (0, 1e4, 0, 1, 1, 2, 100), (257, 1e4, 0, 1, 1, 2, 100), (8, 1.0, 0, 1, 1, 2, 100), (8, math.nan, 0, 1, 1, 2, 100),
    (8, 1e4, 4, 1, 1, 2, 100), (8, 1e4, 1, 0, 1, 2, 100), (8, 1e4, 2, 2, 2, 2, 100), (8, 1e4, 3, 2, 0, 2, 100),
    (8, 1e4, 3, 2, 1, 2, 0),
])
def test_rope_frequencies_refused(args):
    with pytest.raises(vrs.VrsError):
        vrs.rope_freqs(*args)
    assert vrs.lib().vrs_rope_freqs(8, 1e4, 0, 1, 1, 2, 100, None) == -1


# ---- attention ------------------------------------------------------------------------


def attention(ctx, q=FAKE, k=2 * FAKE, v=3 * FAKE, out=4 * FAKE, ws=None, ws_bytes=0,
              seqs=vrs.Seqs(FAKE, None, None, 1, 0, 0), **kw):
    d = vrs.AttentionDesc(q_rows=4, k_rows=4, heads=2, kv_heads=1, head_dim=64, dtype=vrs.BF16, causal=1, scale=0.0,
                          q_ld=128, q_hd=64, k_ld=64, k_hd=64, v_ld=64, v_hd=64, o_ld=128, o_hd=64)
    for key, val in kw.items():
        setattr(d, key, val)
    s = C.byref(seqs) if seqs is not None else None
    return _code(vrs.lib().vrs_attention(ctx, C.byref(d), s, q, k, v, out, ws, ws_bytes, None))


BIG = dict(q_rows=1, k_rows=10000, seqs=vrs.Seqs(FAKE, FAKE, FAKE, 1, 1, 10000))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(out=None)), (-1, dict(seqs=None)),
    (-2, dict(q=FAKE + 8)), (-2, dict(v=FAKE + 2)), (-3, dict(dtype=2)), (-3, dict(head_dim=4)), (-3, dict(head_dim=60)),
    (-3, dict(head_dim=136)), (-2, dict(heads=3, kv_heads=2)), (-2, dict(heads=0)), (-2, dict(kv_heads=0)),
    (-2, dict(q_rows=-1)), (-2, dict(k_rows=-1)), (-1, dict(scale=-0.5)), (-1, dict(scale=math.nan)),
    (-1, dict(scale=math.inf)), (-2, dict(q_ld=132)), (-2, dict(k_hd=60)), (-2, dict(v_ld=-64)),
    (-3, dict(k_ld=1 << 22)), (-2, dict(o_ld=32)), (-2, dict(o_hd=0)), (-2, dict(o_ld=64)),
    (-2, dict(q_hd=1 << 41)), (-1, dict(out=2 * FAKE)), (-1, dict(out=3 * FAKE)),
    (-1, dict(out=FAKE, q_ld=256)), (-1, dict(seqs=vrs.Seqs(None, None, None, 1, 0, 0))),
    (-2, dict(seqs=vrs.Seqs(FAKE, None, None, -1, 0, 0))), (-1, dict(seqs=vrs.Seqs(FAKE, None, None, 1, -1, 0))),
    (-1, dict(BIG)), (-1, dict(BIG, ws=FAKE, ws_bytes=100)), (-1, dict(BIG, ws=FAKE + 4, ws_bytes=1 << 30)),
])
def test_attention_refuses(ctx, code, kw):
    rc, msg = attention(ctx, **kw)
    assert rc == code and "vrs_attention" in msg, (rc, msg)


def test_attention_refuses_keys_past_its_indexes(ctx):
    """Key numbers are int32 and run up to 2^9 past a sequence's last key."""
    rc, msg = attention(ctx, k_rows=(1 << 31) - 512, kv_heads=2)
    assert rc == -3 and "rows" in msg, (rc, msg)
    d = vrs.AttentionDesc(q_rows=1, k_rows=(1 << 31) - 1, heads=4, kv_heads=1, head_dim=64, dtype=vrs.BF16, causal=1, scale=0.0,
                          q_ld=256, q_hd=64, k_ld=64, k_hd=64, v_ld=64, v_hd=64, o_ld=256, o_hd=64)
    size = lambda: vrs.lib().vrs_attention_workspace_size(C.byref(d), C.byref(vrs.Seqs(FAKE, FAKE, FAKE, 1, 1, 0)))   # noqa: E731
    assert size() == 0
    d.k_rows = (1 << 31) - 1024
    assert size() > 0


def test_attention_of_nothing_is_nothing(ctx):
    assert attention(ctx, q_rows=0)[0] == 0
    assert attention(ctx, q_rows=0, q=None, out=None)[0] == 0
    assert attention(ctx, seqs=vrs.Seqs(FAKE, None, None, 0, 0, 0))[0] == 0


def test_wrappers_check_tensors():
    """The binding refuses what the addresses alone would not show."""
    import torch
    c = object.__new__(vrs.Context)
    c.handle, c.device = None, 0
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="context's device"):
        c.rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="contiguous"):
        c.rms_norm(torch.zeros(64, 4).t(), torch.ones(64))
    with pytest.raises(ValueError, match="dtype"):
        c.rms_norm(x.half(), torch.ones(64))
    i = torch.zeros(3, dtype=torch.int32)
    assert vrs.seqs(i).n == 2
    c.device = -1                      # stands for a context on the tensors' device, then for another
    t = torch.zeros(2, 1, 64)
    s = vrs.seqs(i)
    assert c._seqs("x", s) == s.address
    c.device = 0
    with pytest.raises(ValueError, match="context's device"):
        c._seqs("x", s)
    with pytest.raises(ValueError, match="context's device"):
        c.attention(t, t, t, s)
    with pytest.raises(ValueError, match="context's device"):
        c.rope(t, t, torch.zeros(32, dtype=torch.float64))
    for bad in ((i.long(),), (i[:0],), (i, i), (i, i[:2], i), (torch.zeros(6, dtype=torch.int32)[::2],)):
        with pytest.raises(ValueError):
            vrs.seqs(*bad)


def test_packed_descriptors_have_the_structures_layout():
    """The binding packs descriptors as bytes: every field at its place in the C structure."""
    rms_d = vrs.RmsDesc(1, 2, 3, 4, 5, 0.5, 0.25, 6, 7, 8, 9)
    assert vrs._RMS(1, 2, 3, 4, 5, 0.5, 0.25, 6, 7, 8, 9) == bytes(rms_d)
    rope_d = vrs.RopeDesc(1, 2, 3, 4, 5, 6, 7, 8, 9, (C.c_int32 * 4)(10, 11, 12, 13), 0.5, *range(14, 27))
    assert vrs._ROPE(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 0.5, *range(14, 27)) == bytes(rope_d)
    att_d = vrs.AttentionDesc(1, 2, 3, 4, 5, 6, 7, 0.5, *range(8, 16))
    assert vrs._ATTENTION(1, 2, 3, 4, 5, 6, 7, 0.5, *range(8, 16)) == bytes(att_d)


def test_workspace_of_more_sequences_than_an_int_counts_groups():
    """Sequences times key heads past 2^31: split as any other that fill the card, in four parts."""
    d = vrs.AttentionDesc(q_rows=1, k_rows=1 << 20, heads=4, kv_heads=4, head_dim=64, dtype=vrs.BF16, causal=1, scale=0.0,
                          q_ld=256, q_hd=64, k_ld=256, k_hd=64, v_ld=256, v_hd=64, o_ld=256, o_hd=64)
    size = lambda n: vrs.lib().vrs_attention_workspace_size(C.byref(d), C.byref(vrs.Seqs(FAKE, FAKE, FAKE, n, 1, 1 << 20)))   # noqa: E731
    assert size(1 << 20) == size(1 << 30) == 4 * 4 * (64 + 2) * 4

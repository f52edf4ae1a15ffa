"""CPU-side checks of the operators that generate from a cache: what they refuse,
before any HIP call."""
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


def fill(d, kw):
    for key, val in kw.items():
        setattr(d, key, val)
    return d


# ---- attention over shared prefixes -------------------------------------------------

SEQS = vrs.Seqs(FAKE, FAKE, FAKE, 3, 0, 0)
PREFIXES = vrs.Prefixes(FAKE, FAKE, FAKE, 2, 0, 0)


def prefix(ctx, q=FAKE, k=2 * FAKE, v=3 * FAKE, out=4 * FAKE, ws=16 * FAKE, ws_bytes=1 << 40, seqs=SEQS, prefixes=PREFIXES, **kw):
    d = fill(vrs.AttentionDesc(q_rows=4, k_rows=4, heads=2, kv_heads=1, head_dim=64, dtype=vrs.BF16, causal=1, scale=0.0,
                               q_ld=128, q_hd=64, k_ld=64, k_hd=64, v_ld=64, v_hd=64, o_ld=128, o_hd=64), kw)
    ref = [C.byref(x) if x is not None else None for x in (seqs, prefixes)]
    return _code(vrs.lib().vrs_prefix_attention(ctx, C.byref(d), *ref, q, k, v, out, ws, ws_bytes, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(out=None)), (-1, dict(seqs=None)), (-1, dict(prefixes=None)),
    (-2, dict(q=FAKE + 8)), (-3, dict(dtype=2)), (-3, dict(head_dim=60)), (-2, dict(heads=3, kv_heads=2)), (-2, dict(q_ld=132)),
    (-2, dict(o_ld=32)), (-1, dict(out=2 * FAKE)), (-1, dict(out=FAKE, q_ld=256)), (-3, dict(k_rows=(1 << 31) - 512)),
    (-1, dict(ws=None)), (-1, dict(ws_bytes=100)), (-1, dict(ws=FAKE + 4)),
    (-2, dict(prefixes=vrs.Prefixes(FAKE, FAKE, FAKE, -1, 0, 0))), (-1, dict(prefixes=vrs.Prefixes(None, FAKE, FAKE, 1, 0, 0))),
    (-1, dict(prefixes=vrs.Prefixes(FAKE, None, FAKE, 1, 0, 0))), (-1, dict(prefixes=vrs.Prefixes(FAKE, FAKE, None, 1, 0, 0))),
    (-2, dict(prefixes=vrs.Prefixes(FAKE + 2, FAKE, FAKE, 1, 0, 0))), (-1, dict(prefixes=vrs.Prefixes(FAKE, FAKE, FAKE, 1, -1, 0))),
    (-1, dict(prefixes=vrs.Prefixes(FAKE, FAKE, FAKE, 1, 0, -1))), (-2, dict(seqs=vrs.Seqs(FAKE, FAKE, FAKE, -1, 0, 0))),
])
def test_prefix_attention_refuses(ctx, code, kw):
    rc, msg = prefix(ctx, **kw)
    assert rc == code and "vrs_prefix_attention" in msg, (rc, msg)


def test_prefix_attention_of_nothing_is_nothing(ctx):
    assert prefix(ctx, q_rows=0)[0] == 0
    assert prefix(ctx, seqs=vrs.Seqs(FAKE, FAKE, FAKE, 0, 0, 0), q=None)[0] == 0
    assert vrs.lib().vrs_prefix_attention_workspace_size(None, None, None) == 0


# ---- beam search ------------------------------------------------------------------------


def select(ctx, logits=FAKE, scores=2 * FAKE, done=None, outs=(3 * FAKE, 4 * FAKE, 5 * FAKE), ws=16 * FAKE, ws_bytes=1 << 40, **kw):
    d = fill(vrs.BeamDesc(batch=2, beams=3, vocab=1000, k=6, dtype=vrs.F32, eos=5, ld=1000), kw)
    return _code(vrs.lib().vrs_beam_select(ctx, C.byref(d), logits, scores, done, *outs, ws, ws_bytes, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(logits=None)), (-2, dict(logits=FAKE + 2)), (-1, dict(scores=None)), (-1, dict(outs=(None, FAKE, FAKE))),
    (-1, dict(outs=(3 * FAKE, 3 * FAKE, 5 * FAKE))), (-1, dict(outs=(3 * FAKE, 4 * FAKE, 4 * FAKE))), (-1, dict(outs=(2 * FAKE, 4 * FAKE, 5 * FAKE))),
    (-3, dict(dtype=2)), (-2, dict(batch=-1)), (-2, dict(beams=0)), (-3, dict(beams=65)), (-2, dict(vocab=0)), (-2, dict(k=0)),
    (-3, dict(k=129)), (-2, dict(vocab=1, k=4)), (-2, dict(ld=-5)), (-3, dict(beams=64, vocab=1 << 26)), (-3, dict(batch=65535)),
    (-1, dict(done=FAKE, eos=-1)), (-1, dict(done=FAKE, eos=1000)), (-1, dict(ws=None)), (-1, dict(ws_bytes=64)), (-1, dict(ws=FAKE + 8)),
])
def test_beam_select_refuses(ctx, code, kw):
    rc, msg = select(ctx, **kw)
    assert rc == code and "vrs_beam_select" in msg, (rc, msg)


def test_beam_select_of_nothing_is_nothing(ctx):
    assert select(ctx, batch=0, logits=None, scores=None)[0] == 0
    assert vrs.lib().vrs_beam_select_workspace_size(None) == 0
    assert vrs.lib().vrs_beam_select(ctx, None, *[None] * 7, 0, None) == -1


def reorder(ctx, parents=FAKE, lens=None, state=2 * FAKE, **kw):
    d = fill(vrs.ReorderDesc(batch=2, beams=3, layers=4, rows=5, row_bytes=32, row_ld=32, slot_ld=160, layer_ld=960), kw)
    return _code(vrs.lib().vrs_beam_reorder(ctx, C.byref(d), parents, lens, state, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(parents=None)), (-1, dict(state=None)), (-2, dict(parents=FAKE + 2)), (-2, dict(lens=FAKE + 1)), (-2, dict(batch=-1)),
    (-2, dict(beams=0)), (-3, dict(beams=65)), (-2, dict(rows=-1)), (-2, dict(layers=-1)), (-2, dict(row_bytes=-1)), (-2, dict(row_ld=16)),
    (-2, dict(slot_ld=128)), (-2, dict(layer_ld=800)), (-2, dict(layer_ld=-960)), (-2, dict(slot_ld=1 << 43)), (-3, dict(batch=70000, layers=1)),
])
def test_beam_reorder_refuses(ctx, code, kw):
    rc, msg = reorder(ctx, **kw)
    assert rc == code and "vrs_beam_reorder" in msg, (rc, msg)


def test_beam_reorder_of_nothing_is_nothing(ctx):
    for kw in (dict(batch=0), dict(layers=0), dict(rows=0), dict(row_bytes=0)):
        assert reorder(ctx, parents=None, state=None, **kw)[0] == 0


# ---- attention that keys receive ------------------------------------------------------------


def weights(ctx, q=FAKE, k=2 * FAKE, acc=3 * FAKE, ws=16 * FAKE, ws_bytes=1 << 40, seqs=SEQS, **kw):
    d = fill(vrs.WeightsDesc(q_rows=4, k_rows=4, heads=2, kv_heads=1, head_dim=64, dtype=vrs.BF16, causal=1, scale=0.0, decay=1.0,
                             q_ld=128, q_hd=64, k_ld=64, k_hd=64, acc_ld=1, acc_hd=4), kw)
    return _code(vrs.lib().vrs_attention_weights(ctx, C.byref(d), C.byref(seqs) if seqs is not None else None, q, k, acc, ws, ws_bytes, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(acc=None)), (-1, dict(seqs=None)), (-2, dict(q=FAKE + 8)), (-2, dict(acc=FAKE + 2)),
    (-3, dict(dtype=2)), (-3, dict(head_dim=60)), (-3, dict(head_dim=136)), (-2, dict(heads=3, kv_heads=2)), (-2, dict(q_rows=-1)),
    (-2, dict(k_rows=-1)), (-3, dict(k_rows=(1 << 31) - 512)), (-1, dict(scale=-1.0)), (-1, dict(decay=-0.1)), (-1, dict(decay=1.5)),
    (-1, dict(decay=math.nan)), (-2, dict(q_ld=132)), (-2, dict(acc_ld=0)), (-2, dict(acc_ld=-1)), (-2, dict(heads=2, kv_heads=2, acc_hd=0)),
    (-1, dict(acc=FAKE)), (-1, dict(acc=2 * FAKE)), (-1, dict(ws=None)), (-1, dict(ws_bytes=8)), (-1, dict(ws=FAKE + 4)),
    (-3, dict(k_ld=1 << 22)),
])
def test_attention_weights_refuses(ctx, code, kw):
    rc, msg = weights(ctx, **kw)
    assert rc == code and "vrs_attention_weights" in msg, (rc, msg)


def test_attention_weights_of_nothing_is_nothing(ctx):
    assert weights(ctx, k_rows=0, k=None, acc=None)[0] == 0
    assert weights(ctx, seqs=vrs.Seqs(FAKE, FAKE, FAKE, 0, 0, 0), q=None)[0] == 0


# ---- eviction ----------------------------------------------------------------------------------


def evict(ctx, at=FAKE, lens=2 * FAKE, o_start=None, k=3 * FAKE, v=4 * FAKE, acc=5 * FAKE, ko=3 * FAKE, vo=4 * FAKE, ao=5 * FAKE,
          len_out=2 * FAKE, kept=6 * FAKE, **kw):
    d = fill(vrs.EvictDesc(n=2, k_rows=40, out_rows=40, kv_heads=2, head_dim=64, dtype=vrs.BF16, budget=8, first=2, recent=2, max_k=0,
                           k_ld=128, k_hd=64, v_ld=128, v_hd=64, acc_ld=1, acc_hd=40, ko_ld=128, ko_hd=64, vo_ld=128, vo_hd=64,
                           acco_ld=1, acco_hd=40), kw)
    return _code(vrs.lib().vrs_cache_evict(ctx, C.byref(d), at, lens, o_start, k, v, acc, ko, vo, ao, len_out, kept, None))


@pytest.mark.parametrize("code,kw", [
    (-1, dict(at=None)), (-1, dict(lens=None)), (-1, dict(k=None)), (-1, dict(v=None)), (-1, dict(acc=None)), (-1, dict(ko=None)),
    (-1, dict(vo=None)), (-1, dict(ao=None)), (-1, dict(kept=None)), (-2, dict(kept=6 * FAKE + 2)), (-2, dict(k=3 * FAKE + 1)),
    (-3, dict(dtype=2)), (-2, dict(n=-1)), (-2, dict(k_rows=-1)), (-2, dict(out_rows=-1)), (-2, dict(kv_heads=0)), (-2, dict(head_dim=0)),
    (-2, dict(head_dim=5000)), (-1, dict(budget=0)), (-1, dict(first=-1)), (-1, dict(recent=-1)), (-1, dict(first=5, recent=4)),
    (-1, dict(max_k=-1)), (-2, dict(k_ld=-1)), (-2, dict(ko=7 * FAKE, ko_ld=32)), (-2, dict(ko=7 * FAKE, ko_hd=32)), (-2, dict(ko_ld=256)),
    (-2, dict(vo_hd=128, vo_ld=256)), (-2, dict(acco_hd=80)), (-2, dict(o_start=9 * FAKE)), (-2, dict(ao=8 * FAKE, acco_ld=0)),
    (-1, dict(vo=3 * FAKE)), (-1, dict(ko=4 * FAKE)), (-1, dict(len_out=FAKE)), (-1, dict(len_out=6 * FAKE)), (-3, dict(k_rows=(1 << 31) - 512)), (-3, dict(k_rows=(1 << 31) - 2000)), (-3, dict(budget=(1 << 31) - 1)),
])
def test_cache_evict_refuses(ctx, code, kw):
    rc, msg = evict(ctx, **kw)
    assert rc == code and "vrs_cache_evict" in msg, (rc, msg)


def test_cache_evict_of_nothing_is_nothing(ctx):
    assert evict(ctx, n=0, at=None, k=None, kept=None)[0] == 0


def test_cache_evict_addresses_of_empty_buffers_are_of_no_account(ctx):
    """Neither their alignment nor their strides choose a kernel; the calls end at the grid's limit, before a launch."""
    for kw in (dict(k_rows=0, k=3 * FAKE + 2, ko=7 * FAKE, vo=8 * FAKE, ao=9 * FAKE), dict(k_rows=0, v=4 * FAKE + 1, ko=7 * FAKE, vo=8 * FAKE, ao=9 * FAKE),
               dict(out_rows=0, ko=7 * FAKE + 2, vo=8 * FAKE, ao=9 * FAKE), dict(k_rows=0, out_rows=0, k=FAKE + 1, ko=FAKE + 1)):
        rc, msg = evict(ctx, dtype=vrs.F32, n=1 << 21, **kw)
        assert rc == -2 and "grid too large" in msg, (rc, msg, kw)


def test_outputs_that_are_other_arrays_are_refused(ctx):
    """The kernels read what they would write: starts of keys, parents, lengths, logits."""
    for kw in (dict(outs=(3 * FAKE, FAKE, 5 * FAKE)), dict(outs=(3 * FAKE, 4 * FAKE, FAKE)), dict(outs=(3 * FAKE, 2 * FAKE, 5 * FAKE)),
               dict(outs=(3 * FAKE, 4 * FAKE, 2 * FAKE)), dict(done=5 * FAKE), dict(done=4 * FAKE), dict(done=3 * FAKE)):
        rc, msg = select(ctx, **kw)
        assert rc == -1 and "vrs_beam_select: an output" in msg, (rc, msg, kw)
    for kw in (dict(parents=2 * FAKE), dict(lens=2 * FAKE)):
        rc, msg = reorder(ctx, **kw)
        assert rc == -1 and "vrs_beam_reorder: the state" in msg, (rc, msg, kw)
    for kept in (FAKE, 2 * FAKE, 3 * FAKE, 4 * FAKE, 5 * FAKE, 9 * FAKE):
        for kw in ({}, dict(o_start=9 * FAKE, ko=7 * FAKE, vo=8 * FAKE, ao=10 * FAKE)):
            if kept != 9 * FAKE or kw:
                rc, msg = evict(ctx, kept=kept, **kw)
                assert rc == -1 and "vrs_cache_evict: kept is" in msg, (rc, msg, kept, kw)
    for len_out in (3 * FAKE, 5 * FAKE, 7 * FAKE):
        rc, msg = evict(ctx, len_out=len_out, ko=7 * FAKE, vo=8 * FAKE, ao=10 * FAKE)
        assert rc == -1 and "vrs_cache_evict: len_out is" in msg, (rc, msg, len_out)
    for kw in (dict(ao=3 * FAKE), dict(ao=4 * FAKE), dict(ko=7 * FAKE, ao=7 * FAKE), dict(ko=5 * FAKE, ao=7 * FAKE)):
        rc, msg = evict(ctx, **kw)
        assert rc == -1 and "vrs_cache_evict: acc is" in msg, (rc, msg, kw)


# ---- the binding ---------------------------------------------------------------------------------


def test_wrappers_check_tensors():
    import torch
    c = object.__new__(vrs.Context)
    c.handle, c.device = None, 0
    i = torch.zeros(3, dtype=torch.int32)
    t, s = torch.zeros(2, 1, 64), vrs.seqs(i)
    p = vrs.prefixes(i[:2], i[:1], i[:1])
    assert p.n == 1
    for bad in ((i.long(), i[:2], i[:2]), (i[:0], i[:0], i[:0]), (i, i, i[:2]), (torch.zeros(6, dtype=torch.int32)[::2], i[:2], i[:2])):
        with pytest.raises(ValueError):
            vrs.prefixes(*bad)
    for call in (lambda: c.prefix_attention(t, t, t, s, p), lambda: c.attention_weights(t, t, s, torch.zeros(1, 2)),
                 lambda: c.cache_evict(t, t, torch.zeros(1, 2), i[:1], i[:1], 1), lambda: c.beam_select(t, torch.zeros(2, 1), 2),
                 lambda: c.beam_reorder(t, i[:1][None])):
        with pytest.raises(ValueError, match="context's device"):
            call()
    with pytest.raises(ValueError, match="batch, beams, vocab"):
        c.beam_select(torch.zeros(4, 8), torch.zeros(2, 2), 2)
    with pytest.raises(ValueError, match="parents"):
        c.beam_reorder(t, i)


def test_packed_descriptors_have_the_structures_layout():
    assert vrs._BEAM(1, 2, 3, 4, 5, 6, 7) == bytes(vrs.BeamDesc(1, 2, 3, 4, 5, 6, 7))
    assert vrs._REORDER(*range(1, 9)) == bytes(vrs.ReorderDesc(*range(1, 9)))
    assert vrs._WEIGHTS(1, 2, 3, 4, 5, 6, 7, 0.5, 0.25, *range(10, 16)) == bytes(vrs.WeightsDesc(1, 2, 3, 4, 5, 6, 7, 0.5, 0.25, *range(10, 16)))
    assert vrs._EVICT(*range(1, 23)) == bytes(vrs.EvictDesc(*range(1, 23)))

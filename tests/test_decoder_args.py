"""CPU: what the entry points for attention weights, eviction, beams and rotations of several axes refuse, before any
device call.  Handles are stand-ins with the fields that the checks read."""
import ctypes as C

import pytest
import torch

from klearu_amd import _lib
from test_paged_args import ARG, CAP, P, cache, change, refused

NAN, INF = float("nan"), float("inf")


def sections(*n):
    return (C.c_int32 * len(n))(*n)


def test_rope_create_axes():
    out = C.c_void_p()
    base = dict(rot=64, max_pos=100, layout=0, theta=1e4, scaling=0, factor=1.0, orig=0, low=1.0, high=32.0, mag=1.0, axes=3,
                sec=sections(8, 12, 12), restart=0, out=C.byref(out))
    for kw, text in ((dict(axes=0), "axes"), (dict(axes=5), "axes"), (dict(sec=None), "null"), (dict(sec=sections(8, 12, 13)), "sections"),
                     (dict(sec=sections(8, 24, 0)), "section"), (dict(sec=sections(20, 24, -12)), "section"), (dict(axes=2), "sections"),
                     (dict(rot=62), "sections"), (dict(rot=63), "rot_dim"), (dict(rot=1026), "rot_dim"), (dict(out=None), "null"),
                     (dict(scaling=2, factor=2.0, restart=1, sec=sections(1, 15, 16)), "changed base")):
        refused("kh_rope_create_axes", change(base, **kw), ARG, text)


def test_weights():
    base = dict(c=cache(), dtype=0, q=P, qs=256, qh=64, nh=4, rows=3, off=P, batch=3, len=P, table=P, cols=4, ts=4,
                max_rows=1, max_len=64, scale=0.1, causal=1, window=0, lse=P, acc=P, acols=64, ws=None, wsb=0, st=None)
    for kw, text in ((dict(c=None), "null handle"), (dict(dtype=1), "dtype"), (dict(nh=3), "multiple"), (dict(nh=1), "multiple"),
                     (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"), (dict(rows=2 ** 30), "rows"), (dict(batch=-1), "batch"),
                     (dict(cols=0, ts=1), "columns"), (dict(ts=3), "columns"), (dict(cols=2 ** 27, ts=2 ** 27), "positions"),
                     (dict(cols=2 ** 60, ts=2 ** 60), "positions"), (dict(scale=0.0), "scale"), (dict(scale=NAN), "scale"),
                     (dict(scale=3e38), "scale"), (dict(window=-1), "window"), (dict(window=5, causal=0), "window"),
                     (dict(qs=-1), "negative"), (dict(qh=-1), "negative"), (dict(acols=0), "columns"), (dict(q=None), "null"),
                     (dict(off=None), "null"), (dict(len=None), "null"), (dict(table=None), "null"), (dict(lse=None), "null"),
                     (dict(acc=None), "null"), (dict(max_len=-1), "max_len"), (dict(max_rows=-1), "max_rows")):
        refused("kh_paged_kv_weights", change(base, **kw), ARG, text)
    lib = _lib.load()
    for kw in (dict(rows=0, q=None, lse=None), dict(batch=0)):
        assert lib.kh_paged_kv_weights(*change(base, **kw)) == 0
    need = C.c_int64(-1)
    for dtype, rows, batch, most, length in ((0, 3, 3, 1, 64), (2, 5000, 3, 5000, 2 ** 63 - 1), (2, 0, 0, 0, 0),
                                             (2, 2 ** 29, 1, 2 ** 63 - 1, 2 ** 63 - 1), (0, 700, 1, 700, 2 ** 31)):
        assert lib.kh_paged_kv_weights_workspace(cache(), dtype, rows, batch, 4, most, length, C.byref(need)) == 0
        assert 0 <= need.value < 2 ** 48
        if need.value:
            got = dict(dtype=dtype, rows=rows, batch=batch, max_rows=most, max_len=length, ws=P)
            refused("kh_paged_kv_weights", change(base, **got, wsb=need.value - 1), CAP, "workspace")
            refused("kh_paged_kv_weights", change(base, **{**got, "ws": P + 4}, wsb=need.value), ARG, "aligned")
    refused("kh_paged_kv_weights_workspace", (cache(), 0, 3, 3, 4, 1, 64, None), ARG, "null")


def test_evict():
    base = dict(c=cache(), acc=P, acols=100, len=P, batch=2, table=P, cols=8, ts=8, keep=40, recent=10, first=4, kept=P,
                out=P, left=2 * P, ws=P, wsb=1 << 40, st=None)
    for kw, text in ((dict(c=None), "null handle"), (dict(acols=0), "columns"), (dict(acols=2 ** 31), "columns"),
                     (dict(batch=-1), "batch"), (dict(batch=2 ** 31), "batch"), (dict(cols=0, ts=0), "columns"), (dict(ts=7), "columns"),
                     (dict(cols=2 ** 27, ts=2 ** 27), "positions"), (dict(keep=0), "keep"), (dict(keep=-3), "keep"),
                     (dict(keep=2 ** 31), "keep"), (dict(recent=-1), "first"), (dict(first=-1), "first"), (dict(recent=41), "kept"),
                     (dict(first=31), "kept"), (dict(recent=2 ** 62), "kept"), (dict(first=2 ** 62), "kept"), (dict(acc=None), "null"),
                     (dict(len=None), "null"), (dict(table=None), "null"), (dict(kept=None), "null"), (dict(out=None), "null"),
                     (dict(left=None), "null"), (dict(left=P), "place of their own"), (dict(ws=P + 8), "aligned")):
        refused("kh_paged_kv_evict", change(base, **kw), ARG, text)
    # a long sequence's rows go through the workspace, a short one's through registers
    need, lib = C.c_int64(), _lib.load()
    assert lib.kh_paged_kv_evict_workspace(cache(), 2, 40, 100000, C.byref(need)) == 0 and need.value > 0
    refused("kh_paged_kv_evict", change(base, acols=100000, wsb=need.value - 1), CAP, "workspace")
    refused("kh_paged_kv_evict", change(base, acols=100000, ws=None), CAP, "workspace")
    for keep, cols in ((40, 100), (100, 100), (2 ** 31 - 1, 100)):
        assert lib.kh_paged_kv_evict_workspace(cache(), 2, keep, cols, C.byref(need)) == 0 and need.value == 0
    for keep, cols in ((2 ** 31 - 1, 2 ** 31 - 65), (1, 2 ** 31 - 65), (2 ** 31 - 65, 2 ** 31 - 65)):
        assert lib.kh_paged_kv_evict_workspace(cache(), 2 ** 31 - 1, keep, cols, C.byref(need)) == 0 and need.value >= 0
    refused("kh_paged_kv_evict_workspace", (cache(), 2, 0, 100, C.byref(need)), ARG, "keep")
    assert lib.kh_paged_kv_evict(*change(base, batch=0, acc=None)) == 0


def test_reorder():
    base = dict(c=cache(), table=P, cols=8, ts=8, len=P, batch=2, beams=4, parent=P, out=2 * P, os=8, st=None)
    for kw, text in ((dict(c=None), "null handle"), (dict(beams=0), "beams"), (dict(beams=65), "beams"), (dict(batch=-1), "batch"),
                     (dict(batch=2 ** 29), "batch"), (dict(cols=0, ts=0), "columns"), (dict(ts=7), "columns"), (dict(os=7), "apart"),
                     (dict(cols=2 ** 27, ts=2 ** 27, os=2 ** 27), "positions"), (dict(table=None), "null"), (dict(len=None), "null"),
                     (dict(parent=None), "null"), (dict(out=None), "null"), (dict(out=P), "place of its own")):
        refused("kh_paged_kv_reorder", change(base, **kw), ARG, text)
    assert _lib.load().kh_paged_kv_reorder(*change(base, batch=0, table=None)) == 0


def test_select():
    base = dict(dtype=0, x=P, rs=100, batch=2, beams=4, vocab=100, scores=P, done=P, end=2, k=8, y=P, i=P, v=P, ws=P, wsb=1 << 40,
                st=None)
    for kw, text in ((dict(dtype=1), "dtype"), (dict(rs=-1), "negative"), (dict(batch=-1), "batch"), (dict(beams=0), "beams"),
                     (dict(beams=65), "beams"), (dict(vocab=0), "vocab"), (dict(vocab=2 ** 24 + 1), "vocab"), (dict(k=0), "k 0"),
                     (dict(k=65), "k 65"), (dict(vocab=1, k=5), "k 5"), (dict(end=-1), "end"), (dict(end=100), "end"), (dict(x=P + 2), "aligned"),
                     (dict(x=None), "null"), (dict(scores=None), "null"), (dict(y=None), "null"), (dict(i=None), "null"),
                     (dict(v=None), "null"), (dict(ws=P + 8), "aligned")):
        refused("kh_beam_select", change(base, **kw), ARG, text)
    need, lib = C.c_int64(), _lib.load()
    assert lib.kh_beam_select_workspace(2, 4, 100, 8, C.byref(need)) == 0 and need.value > 0
    refused("kh_beam_select", change(base, wsb=need.value - 1), CAP, "workspace")
    refused("kh_beam_select", change(base, ws=None), CAP, "workspace")
    refused("kh_beam_select_workspace", (2, 4, 100, 8, None), ARG, "null")
    assert lib.kh_beam_select(*change(base, batch=0, x=None)) == 0


def test_python_checks_without_a_gpu():
    from klearu_amd import beam, paged
    with pytest.raises(ValueError, match="GPU"):
        beam.select(torch.zeros(1, 2, 5), torch.zeros(1, 2), 2)
    with pytest.raises(ValueError, match="sections"):
        paged.Rope(64, 10, sections=(2 ** 32 + 32,))

"""CPU: what the rotary, paged-cache and paged-attention entry points refuse, before any device call.  Handles
are stand-ins with the fields that the checks read."""
import ctypes as C

import pytest

from klearu_amd import _lib

P = 4096  # a pointer that is never followed


class RopeHandle(C.Structure):
    _fields_ = [("rot", C.c_int), ("layout", C.c_int), ("max_pos", C.c_int64), ("device", C.c_int),
                ("table", C.c_void_p), ("err", C.c_void_p)]


class CacheHandle(C.Structure):
    _fields_ = [("nkv", C.c_int), ("d", C.c_int), ("ps", C.c_int), ("ps_log2", C.c_int), ("pages", C.c_int64),
                ("block", C.c_int64), ("device", C.c_int), ("pool", C.c_void_p), ("err", C.c_void_p)]


def rope(rot=64):
    return C.byref(RopeHandle(rot, 0, 100, 0, P, P))


def cache():
    return C.byref(CacheHandle(2, 64, 16, 4, 10, 1280, 0, P, P))


def refused(name, args, code, text):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    assert rc == code, (rc, lib.kh_last_error())
    assert text in lib.kh_last_error().decode(), lib.kh_last_error()


def change(base, **kw):
    d = dict(base)
    for k in kw:
        assert k in d
    return list({**d, **kw}.values())


ARG, UNS, CAP = _lib.KH_ERR_ARG, _lib.KH_ERR_UNSUPPORTED, _lib.KH_ERR_CAPACITY


def test_rope_create():
    out = C.c_void_p()
    base = dict(rot=64, max_pos=100, layout=0, theta=1e4, scaling=0, factor=1.0, orig=0, low=1.0, high=32.0, mag=1.0,
                out=C.byref(out))
    inf = float("inf")
    for kw, text in ((dict(rot=63), "rot_dim"), (dict(rot=0), "rot_dim"), (dict(rot=1026), "rot_dim"),
                     (dict(max_pos=0), "max_pos"), (dict(max_pos=2 ** 31 + 1), "max_pos"), (dict(layout=2), "layout"),
                     (dict(theta=0.0), "theta"), (dict(theta=inf), "theta"), (dict(scaling=4), "scaling"),
                     (dict(scaling=-1), "scaling"), (dict(scaling=1, factor=0.0), "factor"),
                     (dict(scaling=2, factor=inf), "factor"), (dict(scaling=2, rot=2), "rot_dim > 2"),
                     (dict(scaling=3), "original_len"), (dict(scaling=3, orig=10, low=2.0, high=2.0), "low < high"),
                     (dict(mag=0.0), "magnitude"), (dict(mag=float("nan")), "magnitude"), (dict(out=None), "null")):
        refused("kh_rope_create", change(base, **kw), ARG, text)


def test_rope_apply():
    base = dict(r=rope(), dtype=0, x=P, xs=128, xh=64, rows=3, heads=2, dim=64, pos=P, y=2 * P, ys=128, yh=64, tr=0,
                st=None)
    for kw, text in ((dict(r=None), "null handle"), (dict(dtype=1), "dtype"), (dict(dtype=7), "dtype"),
                     (dict(rows=-1), "rows"), (dict(heads=0), "heads"), (dict(dim=62), "head_dim"),
                     (dict(x=None), "null"), (dict(y=None), "null"), (dict(pos=None), "null"), (dict(xs=-1), "negative"),
                     (dict(yh=63), "overlap"), (dict(ys=64), "overlap"), (dict(ys=0), "overlap"),
                     (dict(y=P, xs=256), "in place")):
        refused("kh_rope_apply", change(base, **kw), ARG, text)
    assert _lib.load().kh_rope_apply(*change(base, rows=0, x=None, y=None, pos=None)) == 0


def test_cache_create():
    out = C.c_void_p()
    base = dict(kv=2, dim=64, page=16, pages=4, out=C.byref(out))
    for kw, code, text in ((dict(kv=0), ARG, "num_kv_heads"), (dict(pages=0), ARG, "num_pages"),
                           (dict(pages=2 ** 31), ARG, "num_pages"), (dict(dim=96), UNS, "head_dim"),
                           (dict(page=8), UNS, "page_size"), (dict(page=48), UNS, "page_size"),
                           (dict(page=512), UNS, "page_size"), (dict(out=None), ARG, "null")):
        refused("kh_paged_kv_create", change(base, **kw), code, text)


def test_append_and_gather():
    base = dict(c=cache(), rope=None, dtype=0, k=P, ks=128, kh=64, v=P, vs=128, vh=64, rows=3, off=P, batch=1, start=P,
                pos=None, table=P, cols=4, ts=4, st=None)
    for kw, text in ((dict(c=None), "null handle"), (dict(dtype=1), "dtype"), (dict(rows=-1), "rows"),
                     (dict(batch=-1), "batch"), (dict(k=None), "null"), (dict(v=None), "null"), (dict(off=None), "null"),
                     (dict(start=None), "null"), (dict(table=None), "null"), (dict(cols=0, ts=0), "columns"),
                     (dict(ts=3), "columns"), (dict(ks=-1), "negative"), (dict(vh=-1), "negative"),
                     (dict(pos=P), "without a rotation"), (dict(rope=rope(128)), "rotation takes")):
        refused("kh_paged_kv_append", change(base, **kw), ARG, text)
    assert _lib.load().kh_paged_kv_append(*change(base, rows=0, k=None, v=None)) == 0
    base = dict(c=cache(), dtype=2, rows=3, off=P, batch=1, start=P, table=P, cols=4, ts=4, k=P, v=P, st=None)
    for kw, text in ((dict(c=None), "null handle"), (dict(dtype=1), "dtype"), (dict(k=None), "null"),
                     (dict(v=None), "null"), (dict(k=P + 2), "aligned"), (dict(ts=1), "columns")):
        refused("kh_paged_kv_gather", change(base, **kw), ARG, text)


def test_attention():
    base = dict(c=cache(), dtype=0, q=P, qs=256, qh=64, nh=4, rows=3, off=P, batch=3, len=P, table=P, cols=4, ts=4,
                max_rows=1, max_len=64, scale=0.1, causal=1, window=0, heads=None, nsel=0, out=2 * P, os=256, oh=64,
                lse=None, ws=None, wsb=0, st=None)
    nan, inf = float("nan"), float("inf")
    for kw, text in ((dict(c=None), "null handle"), (dict(dtype=1), "dtype"), (dict(nh=3), "multiple"),
                     (dict(nh=1), "multiple"), (dict(rows=-1), "rows"), (dict(rows=2 ** 31), "rows"),
                     (dict(cols=0, ts=1), "columns"), (dict(ts=3), "columns"),
                     (dict(cols=2 ** 27, ts=2 ** 27), "positions"), (dict(scale=0.0), "scale"), (dict(scale=nan), "scale"),
                     (dict(scale=inf), "scale"), (dict(scale=-1.0), "scale"), (dict(window=-1), "window"),
                     (dict(window=5, causal=0), "window"), (dict(qs=-1), "negative"), (dict(nsel=17), "n_heads"),
                     (dict(nsel=-1), "n_heads"), (dict(nsel=2), "head list"), (dict(oh=63), "overlap"),
                     (dict(os=128), "overlap"), (dict(q=None), "null"), (dict(off=None), "null"), (dict(len=None), "null"),
                     (dict(table=None), "null"), (dict(out=None), "null"), (dict(max_len=-1), "max_len")):
        refused("kh_paged_kv_attention", change(base, **kw), ARG, text)
    need = C.c_int64()
    call = _lib.load().kh_paged_kv_attention_workspace
    assert call(cache(), 0, 3, 3, 4, 1, 64, 0, C.byref(need)) == 0 and need.value == 0
    assert call(cache(), 0, 3, 3, 4, 1, 100000, 0, C.byref(need)) == 0 and need.value > 0
    refused("kh_paged_kv_attention", change(base, max_len=100000, ws=P, wsb=need.value - 1), CAP, "workspace")
    refused("kh_paged_kv_attention", change(base, max_len=100000), CAP, "workspace")
    refused("kh_paged_kv_attention", change(base, max_len=100000, ws=P + 4, wsb=need.value), ARG, "aligned")
    assert _lib.load().kh_paged_kv_attention(*change(base, rows=0)) == 0


def test_sizes_past_the_types():
    base = dict(r=rope(), dtype=0, x=P, xs=0, xh=64, rows=2 ** 31, heads=2, dim=64, pos=P, y=2 * P, ys=128, yh=64, tr=0,
                st=None)
    refused("kh_rope_apply", list(base.values()), ARG, "rows")
    base = dict(c=cache(), dtype=0, q=P, qs=256, qh=64, nh=4, rows=3, off=P, batch=3, len=P, table=P, cols=4, ts=4,
                max_rows=1, max_len=64, scale=0.1, causal=1, window=0, heads=None, nsel=0, out=2 * P, os=256, oh=64,
                lse=None, ws=None, wsb=0, st=None)
    for kw, text in ((dict(cols=2 ** 60, ts=2 ** 60), "positions"), (dict(scale=3e38), "scale")):
        refused("kh_paged_kv_attention", change(base, **kw), ARG, text)
    need, same = C.c_int64(), C.c_int64()
    call = _lib.load().kh_paged_kv_attention_workspace
    for dtype, rows, most, lse in ((0, 3, 1, 0), (2, 3, 1, 1), (2, 5000, 5000, 0), (2, 5000, 2 ** 62, 1)):
        assert call(cache(), dtype, rows, 3, 4, most, 2 ** 31 - 1, lse, C.byref(need)) == 0
        assert call(cache(), dtype, rows, 3, 4, most, 2 ** 63 - 1, lse, C.byref(same)) == 0
        assert need.value == same.value and (need.value > 0 or rows == 5000)
    assert call(cache(), 2, 2 ** 31 - 1, 2 ** 31 - 1, 2, 2 ** 31 - 1, 2 ** 63 - 1, 1, C.byref(need)) == 0
    assert 0 <= need.value < 2 ** 62

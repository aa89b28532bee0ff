"""Rotary positions, and a paged K/V cache held in 4 bits with the attention that reads it.

The framework's decode step (attention.SparseAttention) keeps a contiguous cache per sequence in
BF16 / f32 and rotates inside the step.  Here the cache is a pool of pages that sequences share,
5 bits a value (include/klearu_hip.h has the format), rows are put in with their rotation on the
way, and attention takes any number of rows per sequence: prompts, chunks of them, single tokens.

    rope = Rope(128, max_pos=32768)
    cache = PagedKv(num_kv_heads=8, head_dim=128, num_pages=4096)
    cache.append(k, v, off, start, table, rope=rope)     # rows off[b]..off[b+1]-1 -> start[b], ...
    q = rope.apply(q, pos)
    y = cache.attention(q, off, start + n_new, table)

All compute runs in libklearu_hip.so on the current torch stream of the tensors' device (or
`stream`).  Rows are tensors [rows, heads, head_dim], f32 or bfloat16, of any non-negative strides
but 1 along the last dimension.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib

HALF, INTERLEAVED = 0, 1
SCALE_NONE, SCALE_LINEAR, SCALE_BASE, SCALE_BY_PARTS = 0, 1, 2, 3

_DT = {torch.float32: 0, torch.bfloat16: 2}
_I64, _I32 = torch.int64, torch.int32


def _elsewhere(t: torch.Tensor, what: str, device: int):
    raise ValueError(f"{what} is on {t.device}, the handle on cuda:{device}")


def _rows(t: torch.Tensor, what: str, device: int, dtype=None):
    """(pointer, row stride, head stride, dtype code) of a tensor [rows, heads, head_dim]."""
    dt = t.dtype
    if t.get_device() != device:
        _elsewhere(t, what, device)
    if t.dim() != 3:
        raise ValueError(f"{what}: expected [rows, heads, head_dim], got {tuple(t.shape)}")
    code = _DT.get(dt)
    if code is None or (dtype is not None and dt is not dtype):
        raise TypeError(f"{what}: dtype {dt}, expected {dtype or 'float32 or bfloat16'}")
    s0, s1, s2 = t.stride()
    if s2 != 1 and t.shape[2] > 1 and t.numel():
        raise ValueError(f"{what}: the elements of a head must be contiguous")
    return t.data_ptr(), s0, s1, code


def _index(t: torch.Tensor, what: str, device: int, dtype, shape):
    """Pointer of a contiguous tensor of a given dtype and shape."""
    if t.get_device() != device:
        _elsewhere(t, what, device)
    if t.dtype is not dtype:
        raise TypeError(f"{what}: dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: expected a contiguous tensor")
    return t.data_ptr()


def _table(t: torch.Tensor, device: int, batch):
    """(pointer, columns, row stride) of an int32 page table [batch, columns]."""
    if t.get_device() != device:
        _elsewhere(t, "table", device)
    if t.dtype is not _I32:
        raise TypeError(f"table: dtype {t.dtype}, expected torch.int32")
    shape = t.shape
    if len(shape) != 2 or shape[0] != batch:
        raise ValueError(f"table: shape {tuple(shape)}, expected [{batch}, columns]")
    cols = shape[1]
    s0, s1 = t.stride()
    if cols > 1 and s1 != 1:
        raise ValueError("table: the columns of a row must be contiguous")
    return t.data_ptr(), cols, max(s0, cols) if batch <= 1 else s0


def _check(rc: int) -> None:
    if rc < 0:
        raise _lib.KlearuError(rc, _lib.load().kh_last_error().decode(errors="replace"))


class _On:
    """Makes a handle's device and `stream` (None: the current one) current, and holds the memory
    of `tensors` for that stream; as a value, the stream's pointer."""

    def __init__(self, device, stream, tensors):
        if stream is not None and stream.device != device:
            raise ValueError(f"stream is on {stream.device}, the handle on {device}")
        self.ctx = [torch.cuda.device(device)]
        if stream is not None:
            self.ctx.append(torch.cuda.stream(stream))
        self.stream, self.tensors = stream, tensors

    def __enter__(self):
        for c in self.ctx:
            c.__enter__()
        if self.stream is not None:
            for t in self.tensors:
                if t is not None:
                    t.record_stream(self.stream)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *e):
        for c in reversed(self.ctx):
            c.__exit__(*e)


# torch.cuda.current_stream(index).cuda_stream and torch.cuda.current_device(), without the
# objects (a call of a few microseconds is mostly this)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda i: torch.cuda.current_stream(i).cuda_stream)
_raw_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


class _Handle:
    _destroy = ""

    def __del__(self):
        h = getattr(self, "_h", None)
        if h:
            try:
                getattr(_lib.load(), self._destroy)(h)
            except Exception:
                pass

    def _adopt(self, h):
        self._h = h
        self._lib = _lib.load()
        self._dev = torch.cuda.current_device()
        self.device = torch.device("cuda", self._dev)

    def _status(self, name):
        with _On(self.device, None, ()):
            _check(getattr(self._lib, name)(self._h))


class Rope(_Handle):
    """Rotation of the first `rot_dim` elements of heads by positions 0 .. max_pos - 1.

    layout HALF rotates element i with i + rot_dim / 2 (crates/klearu-llm/src/model/rope.rs:75-87),
    INTERLEAVED 2 i with 2 i + 1.  Frequencies theta^(-2 i / rot_dim) are stretched for contexts
    longer than the trained one by `factor`: SCALE_LINEAR all of them, SCALE_BASE through theta,
    SCALE_BY_PARTS those that turn less than `low` times over `original_len` positions, those
    over `high` turns not, in between in proportion.  `magnitude` scales the rotated elements."""

    _destroy = "kh_rope_destroy"

    def __init__(self, rot_dim, max_pos, layout=HALF, theta=10000.0, scaling=SCALE_NONE, factor=1.0, original_len=0,
                 low=1.0, high=32.0, magnitude=1.0):
        h = C.c_void_p()
        _lib.call("kh_rope_create", rot_dim, max_pos, layout, theta, scaling, factor, original_len, low, high,
                  magnitude, C.byref(h))
        self._adopt(h)
        self.rot_dim, self.max_pos, self.layout = rot_dim, max_pos, layout

    def apply(self, x: torch.Tensor, pos: torch.Tensor, out: torch.Tensor | None = None, transpose: bool = False,
              stream=None) -> torch.Tensor:
        """x [rows, heads, head_dim] rotated by pos [rows] (int64), into `out` (x itself rotates in
        place) or a new tensor.  `transpose` takes gradients back: the transposed rotation.  Rows of
        a negative position are padding and left as they were, as are (reported by status()) rows
        past max_pos; in a new tensor those hold no value."""
        dev = self._dev
        xp, x0, x1, dt = _rows(x, "x", dev)
        n, heads, dim = x.shape
        pp = _index(pos, "pos", dev, _I64, (n,))
        if stream is not None or _raw_device() != dev:
            with _On(self.device, stream, (x, pos, out)):
                return self.apply(x, pos, out, transpose)
        if out is None:
            out = torch.empty_like(x, memory_format=torch.contiguous_format)
            yp, y0, y1 = out.data_ptr(), heads * dim, dim
        elif out.shape != x.shape:
            raise ValueError(f"out: shape {tuple(out.shape)}, expected {tuple(x.shape)}")
        else:
            yp, y0, y1, _ = _rows(out, "out", dev, x.dtype)
        _check(self._lib.kh_rope_apply(self._h, dt, xp, x0, x1, n, heads, dim, pp, yp, y0, y1, 1 if transpose else 0,
                                       _raw_stream(dev)))
        return out

    def status(self):
        """Raise KlearuError (KH_ERR_ARG) if a call since the last check met a position past max_pos."""
        self._status("kh_rope_status")


class PagedKv(_Handle):
    """num_pages pages of page_size positions of every kv head, keys and values in 4 bits.

    A page table [batch, columns] (int32) names each sequence's pages, and off [batch + 1] (int64)
    the rows of a call that are its own: off[b] .. off[b + 1] - 1.  Rows outside are padding.
    Which page is whose is the caller's; pages may be shared by sequences that only read them."""

    _destroy = "kh_paged_kv_destroy"

    def __init__(self, num_kv_heads, head_dim, num_pages, page_size=64):
        h = C.c_void_p()
        _lib.call("kh_paged_kv_create", num_kv_heads, head_dim, page_size, num_pages, C.byref(h))
        self._adopt(h)
        self.num_kv_heads, self.head_dim = num_kv_heads, head_dim
        self.num_pages, self.page_size = num_pages, page_size
        self._ws = {}

    def _places(self, off, start, table):
        """What every call over rows of sequences checks: (batch, off, start, table, columns, stride)."""
        dev, batch = self._dev, start.shape[0]
        return (batch, _index(off, "off", dev, _I64, (batch + 1,)), _index(start, "start", dev, _I64, (batch,)),
                *_table(table, dev, batch))

    def append(self, k: torch.Tensor, v: torch.Tensor, off: torch.Tensor, start: torch.Tensor, table: torch.Tensor,
               rope: Rope | None = None, pos: torch.Tensor | None = None, stream=None) -> None:
        """Row off[b] + i of k and v [rows, num_kv_heads, head_dim] becomes position start[b] + i of
        sequence b; `rope` rotates the keys on the way, by pos [rows] or by their places in the
        cache.  Two rows of one call must not have the same place."""
        dev = self._dev
        kp, k0, k1, dt = _rows(k, "k", dev)
        vp, v0, v1, _ = _rows(v, "v", dev, k.dtype)
        n = k.shape[0]
        shape = (n, self.num_kv_heads, self.head_dim)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"k, v: shapes {tuple(k.shape)}, {tuple(v.shape)}, expected {shape}")
        batch, op, sp, tp, cols, ts = self._places(off, start, table)
        if pos is not None and rope is None:
            raise ValueError("pos: rotary positions without a rotation")
        pp = None if pos is None else _index(pos, "pos", dev, _I64, (n,))
        if stream is not None or _raw_device() != dev:
            with _On(self.device, stream, (k, v, off, start, table, pos)):
                return self.append(k, v, off, start, table, rope, pos)
        _check(self._lib.kh_paged_kv_append(self._h, None if rope is None else rope._h, dt, kp, k0, k1, vp, v0, v1, n, op,
                                            batch, sp, pp, tp, cols, ts, _raw_stream(dev)))

    def gather(self, off: torch.Tensor, start: torch.Tensor, table: torch.Tensor, rows: int,
               dtype: torch.dtype = torch.float32, k: torch.Tensor | None = None, v: torch.Tensor | None = None,
               stream=None):
        """The values that those places hold: (k, v) [rows, num_kv_heads, head_dim], new or given.
        Rows outside all sequences, or without a place, are left as they were."""
        dev = self._dev
        batch, op, sp, tp, cols, ts = self._places(off, start, table)
        dt = _DT.get(dtype)
        if dt is None:
            raise TypeError(f"dtype {dtype}: expected float32 or bfloat16")
        if stream is not None or _raw_device() != dev:
            with _On(self.device, stream, (off, start, table, k, v)):
                return self.gather(off, start, table, rows, dtype, k, v)
        shape = (rows, self.num_kv_heads, self.head_dim)
        if k is None:
            k = torch.empty_strided(shape, (shape[1] * shape[2], shape[2], 1), dtype=dtype, device=self.device)
            kp = k.data_ptr()
        else:
            kp = _index(k, "k", dev, dtype, shape)
        if v is None:
            v = torch.empty_like(k)
            vp = v.data_ptr()
        else:
            vp = _index(v, "v", dev, dtype, shape)
        _check(self._lib.kh_paged_kv_gather(self._h, dt, rows, op, batch, sp, tp, cols, ts, kp, vp, _raw_stream(dev)))
        return k, v

    def attention(self, q: torch.Tensor, off: torch.Tensor, lens: torch.Tensor, table: torch.Tensor,
                  scale: float | None = None, causal: bool = True, window: int = 0,
                  heads: torch.Tensor | None = None, max_rows: int | None = None, max_len: int | None = None,
                  out: torch.Tensor | None = None, return_lse: bool = False, stream=None):
        """Attention of q [rows, num_heads, head_dim] over the cache: sequence b holds lens[b]
        positions, the last of them its rows' own (append first).  scale defaults to
        head_dim ** -0.5.  heads [rows, n] (int32, SparsityPredictor.select_top_k's lists) leaves
        the other heads 0.  max_rows and max_len guess the most rows and the longest length of a
        sequence (default: an even share of the rows, the table's reach); wrong guesses cost
        time and workspace.  Returns out, or (out, lse) with lse [rows, num_heads] f32: a row that
        sees nothing gives 0 and -inf."""
        dev = self._dev
        qp, q0, q1, dt = _rows(q, "q", dev)
        n, nh, dim = q.shape
        if dim != self.head_dim:
            raise ValueError(f"q: head_dim {dim}, expected {self.head_dim}")
        batch, op, lp, tp, cols, ts = self._places(off, lens, table)
        hp, nsel = None, 0
        if heads is not None:
            nsel = heads.shape[-1]
            hp = _index(heads, "heads", dev, _I32, (n, nsel)) or op  # an empty list is no list of all
        if stream is not None or _raw_device() != dev:
            with _On(self.device, stream, (q, off, lens, table, heads, out)):
                return self.attention(q, off, lens, table, scale, causal, window, heads, max_rows, max_len, out,
                                      return_lse)
        if max_rows is None:
            max_rows = -(-n // max(1, batch))
        if max_len is None:
            max_len = cols * self.page_size
        if scale is None:
            scale = dim ** -0.5
        need = self._workspace(dt, n, batch, nh, max_rows, max_len, 1 if return_lse else 0)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            yp, y0, y1 = out.data_ptr(), nh * dim, dim
        elif out.shape != q.shape:
            raise ValueError(f"out: shape {tuple(out.shape)}, expected {tuple(q.shape)}")
        else:
            yp, y0, y1, _ = _rows(out, "out", dev, q.dtype)
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        lse = torch.empty((n, nh), dtype=torch.float32, device=self.device) if return_lse else None
        _check(self._lib.kh_paged_kv_attention(
            self._h, dt, qp, q0, q1, nh, n, op, batch, lp, tp, cols, ts, max_rows, max_len, scale, 1 if causal else 0,
            window, hp, nsel, yp, y0, y1, None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(),
            need, _raw_stream(dev)))
        return (out, lse) if return_lse else out

    def _workspace(self, *sizes) -> int:
        """kh_paged_kv_attention_workspace: bytes by the call's sizes."""
        need = self._ws.get(sizes)
        if need is None:
            x = C.c_int64()
            _check(self._lib.kh_paged_kv_attention_workspace(self._h, *sizes, C.byref(x)))
            if len(self._ws) >= 1024:
                self._ws.clear()
            need = self._ws[sizes] = x.value
        return need

    def status(self):
        """Raise KlearuError (KH_ERR_ARG) if a call since the last check met a place outside its
        sequence's table, a length the table cannot hold, or a page id outside the pool."""
        self._status("kh_paged_kv_status")

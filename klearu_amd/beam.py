"""Beams: the best continuations of every sequence over beams and vocabulary.

    scores, parent, token = select(logits, scores, k=beams, done=done, end=2)
    table = cache.reorder(table, lens, parent)     # paged.PagedKv: the beams' page tables

klearu has no counterpart.  The compute runs in libklearu_hip.so on the current torch stream of the logits' device (or
`stream`).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from .paged import _DT, _check, _index, _On, _raw_device, _raw_stream

_spaces: dict = {}


def _space(*sizes) -> int:
    need = _spaces.get(sizes)
    if need is None:
        x = C.c_int64()
        _check(_lib.load().kh_beam_select_workspace(*sizes, C.byref(x)))
        if len(_spaces) >= 1024:
            _spaces.clear()
        need = _spaces[sizes] = x.value
    return need


def select(logits: torch.Tensor, scores: torch.Tensor, k: int, done: torch.Tensor | None = None, end: int = 0,
           stream=None):
    """The k best of scores[b, i] + log_softmax(logits[b, i])[v] over the beams i and tokens v of
    each sequence b, best first, of equal ones the first by (i, v).  logits [batch, beams, vocab]
    (f32 or bfloat16; rows may be apart), scores [batch, beams] f32.  A beam that is `done` [batch,
    beams] (bool) has one continuation, the token `end`, at its own score.  Beams whose score is not
    finite have none: at the first step, where all beams are alike, all but one have -inf.  Returns
    (scores f32, beams int32, tokens int32), each [batch, k]; -inf where there are fewer."""
    device = logits.device
    dev = logits.get_device()
    if dev < 0:
        raise ValueError(f"logits is on {device}, expected a GPU")
    dt = _DT.get(logits.dtype)
    if dt is None:
        raise TypeError(f"logits: dtype {logits.dtype}, expected float32 or bfloat16")
    if logits.dim() != 3:
        raise ValueError(f"logits: expected [batch, beams, vocab], got {tuple(logits.shape)}")
    batch, beams, vocab = logits.shape
    s0, s1, s2 = logits.stride()
    if vocab > 1 and s2 != 1:
        raise ValueError("logits: the tokens of a beam must be contiguous")
    if beams == 1:
        s1 = s0
    elif batch > 1 and s0 != beams * s1:
        raise ValueError("logits: sequences must be as far apart as their beams are")
    sp = _index(scores, "scores", dev, torch.float32, (batch, beams))
    dp = None if done is None else _index(done, "done", dev, torch.bool, (batch, beams))
    if stream is not None or _raw_device() != dev:
        with _On(device, stream, (logits, scores, done)):
            return select(logits, scores, k, done, end)
    need = _space(batch, beams, vocab, k)
    y = torch.empty((batch, k), dtype=torch.float32, device=device)
    i = torch.empty((batch, k), dtype=torch.int32, device=device)
    v = torch.empty_like(i)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _check(_lib.load().kh_beam_select(dt, logits.data_ptr(), s1, batch, beams, vocab, sp, dp, end, k, y.data_ptr(), i.data_ptr(),
                                      v.data_ptr(), ws.data_ptr(), need, _raw_stream(dev)))
    return y, i, v

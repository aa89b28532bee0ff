"""GPU: attention over the paged 4-bit cache, each kernel held to its own roundings.

Cases and the plain form are those of test_gpu_paged_attn and paged_ref.  Here a call's tolerance goes by what the
header promises for its sequence: BF16 weights to 2^-16 in sequences (or windows) of 1024 positions or fewer, to 2^-8
past them; keys and values rounded to BF16 in tiles of many rows alone (`many`)."""
import numpy as np
import pytest
import torch

from paged_ref import attention
from test_gpu_paged_attn import BF16, F32, Case

pytestmark = pytest.mark.gpu


def hold(c, got, causal=True, window=0, many=False, on=None):
    """got is `out` or (out, lse) of the case's rows: every element within its own tolerance."""
    out, lse = (None if x is None else x.double().cpu().numpy() for x in ((got, None) if torch.is_tensor(got) else got))
    at = 0
    for n, length, k, v in zip(c.rows, c.lens, c.k, c.v):
        rows, at = slice(at, at + n), at + n
        if n == 0:
            continue
        assert 1 <= n <= length
        fine = not many and min(length, window or length) <= 1024
        o, l, to, tl = attention(c.q[rows].double().numpy(), k.float().numpy(), v.float().numpy(), c.dim ** -0.5, causal,
                                 window, c.dtype == BF16, many, fine)
        if on is not None:
            off = ~on[rows]
            o[off], l[off], to[off], tl[off] = 0, -np.inf, 0, 0
        assert (np.isnan(out[rows]) == np.isnan(o)).all()
        there = ~np.isnan(o)
        d = np.abs(out[rows] - o)
        assert (d[there] <= to[there]).all(), (length, float(np.max(np.where(there, d / np.where(to > 0, to, 1), 0))))
        if lse is not None:
            some = np.isfinite(l)
            assert (np.isnan(lse[rows]) == np.isnan(l)).all()
            assert (lse[rows][~some & ~np.isnan(l)] == -np.inf).all()
            assert (np.abs(lse[rows][some] - l[some]) <= tl[some]).all()
    c.cache.status()


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (8, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("lens,window", [([1, 7, 20, 33, 150, 512, 513], 0), ([1023, 1024, 5], 0), ([1025, 30, 1024, 2100], 0),
                                         ([2000, 900, 31], 24)])
def test_weights_by_the_lengths(kh, heads, kv, dim, lens, window):
    """The bits of a weight go by its sequence, whatever the caller guesses (a table far wider than the lengths)."""
    c = Case(BF16, heads, kv, dim, 32, [1] * len(lens), lens)
    for guess in (None, max(lens), 64, 4096, 10 ** 5):
        hold(c, c.run(window=window, max_len=guess), window=window)
        hold(c, c.run(window=window, max_len=guess, max_rows=1, return_lse=False), window=window)

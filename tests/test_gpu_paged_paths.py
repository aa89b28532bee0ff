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


def hold(c, got, causal=True, window=0, many=False, on=None, seqs=None, heads=None, status=True):
    """got is `out` or (out, lse) of the case's rows: every element within its own tolerance, of all sequences and heads
    or of those given."""
    out, lse = (None if x is None else x for x in ((got, None) if torch.is_tensor(got) else got))
    at = np.concatenate([[0], np.cumsum(c.rows)])
    hs = list(range(c.heads)) if heads is None else heads
    for b in range(len(c.rows)) if seqs is None else seqs:
        n, length, rows = c.rows[b], c.lens[b], slice(at[b], at[b + 1])
        if n == 0:
            continue
        assert 1 <= n <= length
        fine = not many and min(length, window or length) <= 1024
        y = out[rows][:, hs].double().cpu().numpy()
        z = None if lse is None else lse[rows][:, hs].double().cpu().numpy()
        q, k, v = c.q[rows].double().numpy(), c.k[b].float().numpy(), c.v[b].float().numpy()
        for i, h in enumerate(hs):
            g = slice(h * c.kv // c.heads, h * c.kv // c.heads + 1)
            o, l, to, tl = (x[:, 0] for x in attention(q[:, h:h + 1], k[:, g], v[:, g], c.dim ** -0.5, causal, window,
                                                       c.dtype == BF16, many, fine))
            if on is not None:
                off = ~on[rows, h]
                o[off], l[off], to[off], tl[off] = 0, -np.inf, 0, 0
            assert (np.isnan(y[:, i]) == np.isnan(o)).all(), (b, h)
            there = ~np.isnan(o)
            d = np.abs(y[:, i] - o)
            assert (d[there] <= to[there]).all(), (b, length, h, float(np.max(np.where(there, d / np.where(to > 0, to, 1), 0))))
            if z is not None:
                some = np.isfinite(l)
                assert (np.isnan(z[:, i]) == np.isnan(l)).all(), (b, h)
                assert (z[:, i][~some & ~np.isnan(l)] == -np.inf).all(), (b, h)
                assert (np.abs(z[:, i][some] - l[some]) <= tl[some]).all(), (b, h)
    if status:
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


# ---------------------------------------------------------------- positions unpacked ahead (BF16 tiles of many rows)
def unpacked(c, most_rows, most_len, lse):
    """(bytes of unpacked positions, bytes of their masks) where the plan takes that path in one part, as its workspace
    says: steps of 64 positions (32 of 256-wide heads with the log-sum-exp) of values, and of keys in one or two terms,
    and one bit of 32 positions for each group of 32 elements."""
    keys = 32 if c.dim == 256 and lse else 64
    steps = -(-most_len // keys) * len(c.rows) * c.kv
    step, masks = keys * c.dim * 2 * (3 if lse else 2), c.dim // 32 * (keys // 32) * 4
    need = c.cache._workspace(2, sum(c.rows), len(c.rows), c.heads, most_rows, most_len, 1 if lse else 0)
    assert need == steps * (step + masks), (need, steps, step, masks)
    return steps * step, steps * masks


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lse", [False, True])
def test_masks_are_written_whole(kh, dim, lse):
    """No word of a workspace is read that was not written: every mask word of a whole sequence is, and the bits that
    lay there before do not matter."""
    from klearu_amd import _lib
    c = Case(BF16, 512, 4, dim, 64, [210], [704])
    c.v[0][5, 1, 40] = float("nan")
    c.cache.append(c.k[0].cuda(), c.v[0].cuda(), torch.tensor([0, 704]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), c.table)
    data, masks = unpacked(c, 210, 704, lse)
    q, got = c.q.cuda(), []
    for fill in (0x5A, 0x00, 0xFF):
        ws = torch.full((data + masks,), fill, dtype=torch.uint8, device="cuda")
        out = torch.zeros_like(q)
        l = torch.zeros(210, 512, device="cuda") if lse else None
        rc = _lib.load().kh_paged_kv_attention(
            c.cache._h, 2, q.data_ptr(), 512 * dim, dim, 512, 210, c.off.data_ptr(), 1, c.len.data_ptr(), c.table.data_ptr(),
            c.table.shape[1], c.table.shape[1], 210, 704, dim ** -0.5, 1, 0, None, 0, out.data_ptr(), 512 * dim, dim,
            None if l is None else l.data_ptr(), ws.data_ptr(), data + masks, torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        assert (ws[data:].view(torch.int32) != 0x5A5A5A5A).all()
        got.append((out, l))
    for o, l in got[1:]:
        assert torch.equal(o.view(torch.int16), got[0][0].view(torch.int16)) and (l is None or torch.equal(l, got[0][1]))
    assert torch.isnan(got[0][0]).any()


# ---------------------------------------------------------------- grids past a launch's threads
def test_guess_of_the_rows_past_one_grid(kh):
    """1000 sequences of 33 to 35 rows, and every row of the call as the guess of one sequence's: 2^32 threads of tiles."""
    n = [33 + b % 3 for b in range(1000)]
    c = Case(BF16, 64, 8, 64, 16, n, [r + b % 5 for b, r in enumerate(n)])
    want = c.run(max_rows=35, max_len=40)
    hold(c, want, many=True, seqs=[0, 1, 500, 998, 999], heads=[0, 20, 63])
    for guess in (sum(n), 10 ** 6):
        got = c.run(max_rows=guess, max_len=40)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_guess_of_the_rows_of_many_sequences(kh):
    """20000 sequences of two rows, f32, and that guess: more row tiles than a grid's 2^31 blocks."""
    c = Case(F32, 64, 8, 64, 16, [2] * 20000, [2 + b % 4 for b in range(20000)])
    hold(c, c.run(max_rows=40000, max_len=16), seqs=[0, 1, 2, 9999, 19998, 19999], heads=[0, 31, 63])


def test_padding_past_one_grid_of_the_join(kh):
    """One row behind 2^17 rows of padding, in 17 parts: 2^24 + 128 rows of heads to join, 75 GB of workspace."""
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GiB of device memory")
    c = Case(F32, 128, 1, 64, 64, [1], [4352])
    rows = 2 ** 17 + 1
    assert c.cache._workspace(0, rows, 1, 128, 1, 4352, 0) == rows * 128 * 17 * (4 * 64 + 8)
    q = c.q.cuda().expand(rows, 128, 64)
    out = torch.full((rows, 128, 64), 7.0, device="cuda")
    off = torch.tensor([rows - 1, rows], device="cuda")
    c.cache.attention(q, off, c.len, c.table, max_rows=1, max_len=4352, out=out)
    hold(c, out[-1:])
    assert bool((out[:-1] == 7).all())

"""GPU: attention over the paged 4-bit cache, each kernel held to its own roundings.

Cases and the plain form are those of test_gpu_paged_attn and paged_ref.  Here a call's tolerance goes by what the
header promises for its sequence: BF16 weights to 2^-16 in sequences (or windows) of 1024 positions or fewer, to 2^-8
past them; keys and values rounded to BF16 in tiles of many rows alone (`many`)."""
import numpy as np
import pytest
import torch

from paged_ref import attention, offsets, quantize
from test_gpu_paged_attn import BF16, F32, SHAPES, Case

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
def unpacked(c, most_rows, most_len, lse, parts=0):
    """(bytes of unpacked positions, bytes of their masks) where the plan takes that path in one part, or in so many, as
    its workspace says: steps of 64 positions (32 of 256-wide heads with the log-sum-exp) of values, and of keys in one or
    two terms, and one bit of 32 positions for each group of 32 elements."""
    keys = 32 if c.dim == 256 and lse else 64
    steps = -(-most_len // keys) * len(c.rows) * c.kv
    step, masks = keys * c.dim * 2 * (3 if lse else 2), c.dim // 32 * (keys // 32) * 4
    need = c.cache._workspace(2, sum(c.rows), len(c.rows), c.heads, most_rows, most_len, 1 if lse else 0)
    joined = -(-sum(c.rows) * c.heads * parts * (4 * c.dim + 8) // 16) * 16
    assert need == joined + steps * (step + masks), (need, joined, steps, step, masks)
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


def again(c):
    """The case's keys and values appended once more, after a change."""
    c.cache.append(torch.cat(c.k).cuda(), torch.cat(c.v).cuda(), offsets(c.lens).cuda(),
                   torch.zeros(len(c.lens), dtype=torch.int64).cuda(), c.table)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 128])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 70), (False, 0)])
@pytest.mark.parametrize("lse", [False, True])
def test_unpacked_in_one_part(kh, dim, page, causal, window, lse):
    """Whole positions, then groups that stand for NaN; the guess covers every sequence, or all but the longest one."""
    rows, lens, heads = [120, 0, 60, 40], [700, 9, 60, 300], [0, 127, 130, 300, 511]
    c = Case(BF16, 512, 4, dim, page, rows, lens)
    for bad in (False, True):
        if bad:
            c.v[0][690, 1, 40], c.v[0][100, 3, dim - 1] = float("nan"), float("inf")
            c.v[2][30, 0, 33], c.k[3][280, 2, 5] = -float("inf"), float("nan")
            again(c)
        for guess in (704, 640):
            unpacked(c, 120, guess, lse)
            got = c.run(causal=causal, window=window, max_rows=120, max_len=guess, return_lse=lse)
            hold(c, got, causal, window, many=True, heads=heads)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lse", [False, True])
def test_unpacked_in_parts(kh, dim, lse):
    """The same where the positions are cut in three."""
    n = 150 if dim == 256 else 330
    c = Case(BF16, 64, 4, dim, 32, [n], [1500])
    c.v[0][1400, 2, 3], c.v[0][5, 0, 33] = float("nan"), float("nan")
    again(c)
    unpacked(c, n, 3500, lse, parts=3)
    for window in (0, 200):
        got = c.run(max_rows=n, max_len=3500, window=window, return_lse=lse)
        hold(c, got, window=window, many=True, heads=[0, 15, 17, 40, 63])


def without(c, b, first, count):
    """The case as if sequence b had no positions first .. first + count - 1 (all its rows are behind them)."""
    assert first + count <= c.lens[b] - c.rows[b]
    keep = [i for i in range(c.lens[b]) if not first <= i < first + count]
    c.k[b], c.v[b], c.lens[b] = c.k[b][keep], c.v[b][keep], len(keep)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("guess", [800, 2400])
def test_tiles_past_one_round_of_pages(kh, dim, lse, guess):
    """2400 positions in one part, where the tiles hold the pages of 1024 at a time: unpacked by each tile (a guess that
    is too small) and ahead; then pages of the first, second and third round that are not there."""
    from klearu_amd import KlearuError
    c = Case(BF16, 128, 4, dim, 16, [300], [2400])
    if guess == 2400:
        unpacked(c, 300, guess, lse)
    else:
        assert c.cache._workspace(2, 300, 1, 128, 300, guess, 1 if lse else 0) == 0
    heads, most = [0, 31, 33, 80, 127], dict(max_rows=300, max_len=guess, return_lse=lse)
    hold(c, c.run(**most), many=True, heads=heads)
    for at in (2064, 1520, 1024, 1008, 16):
        c.table[0, at // 16] = c.cache.num_pages
        got = c.run(**most)
        with pytest.raises(KlearuError, match="page id"):
            c.cache.status()
        without(c, 0, at, 16)
        hold(c, got, many=True, heads=heads, status=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_single_rows_past_one_round_of_pages(kh, dtype, dim, page):
    """20000 and 17001 positions in one part, where a wave holds the pages of 64 of its steps at a time (8192 or 16384
    positions of the block's); then pages of each round that are not there."""
    from klearu_amd import KlearuError
    c = Case(dtype, 4, 2, dim, page, [1, 3], [20000, 17001])
    assert c.cache._workspace(0 if dtype == F32 else 2, 4, 2, 4, 3, 100, 1) == 0
    hold(c, c.run(max_rows=3, max_len=100))
    for at in (19904, 16384, 8128):
        c.table[0, at // page] = -1
        got = c.run(max_rows=3, max_len=100)
        with pytest.raises(KlearuError, match="page id"):
            c.cache.status()
        without(c, 0, at, page)
        hold(c, got, seqs=[0], heads=[0, 3], status=False)


# ---------------------------------------------------------------- single rows, weights in one term and in two
SHORT = [1, 2, 15, 16, 17, 31, 33, 64, 65, 128, 129, 511, 513, 1023, 1024]
LONG = [1025, 1057, 2048, 2049]


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("lens", [SHORT, LONG])
def test_terms_single_rows(kh, heads, kv, dim, lens):
    c = Case(BF16, heads, kv, dim, 32, [1] * len(lens), lens)
    hold(c, c.run())
    hold(c, c.run(max_len=max(lens), return_lse=False))


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (8, 2, 64), (6, 2, 256), (3, 1, 128), (40, 2, 64)])
@pytest.mark.parametrize("rows,lens", [([3, 1, 2], [3, 700, 1024]), ([1, 3, 2], [1025, 1500, 1060])])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1024), (True, 1025), (True, 5)])
def test_terms_few_rows(kh, heads, kv, dim, rows, lens, causal, window):
    c = Case(BF16, heads, kv, dim, 16, rows, lens)
    hold(c, c.run(causal=causal, window=window), causal, window)
    n, rng = sum(rows), np.random.default_rng(3)
    sel = np.stack([rng.permutation(heads)[: max(1, heads // 3)] for _ in range(n)]).astype(np.int32)
    on = np.zeros((n, heads), bool)
    np.put_along_axis(on, sel.astype(np.int64), True, 1)
    hold(c, c.run(causal=causal, window=window, heads=torch.from_numpy(sel).cuda()), causal, window, on=on)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (4, 2, 128), (6, 2, 256)])
@pytest.mark.parametrize("lens", [[200, 150], [1300, 1200]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_terms_not_finite(kh, dtype, heads, kv, dim, lens, bad):
    """A value's group and a key that are not finite, with rows before and behind them; the same pages with finite rows
    after that, and a shorter sequence over them."""
    c = Case(dtype, heads, kv, dim, 16, [5, 1], list(lens))
    k, v = [x.clone() for x in c.k], [x.clone() for x in c.v]
    c.v[0][lens[0] - 3, 1, 40], c.v[1][3, 0, 0] = bad, bad
    again(c)
    hold(c, c.run())
    hold(c, c.run(window=64), window=64)
    c.k[0][lens[0] - 2, 0, 5] = bad
    again(c)
    hold(c, c.run())
    c.k, c.v = k, v
    again(c)
    hold(c, c.run())
    # the pages' last positions hold NaN, and no sequence reaches them
    c.k[0][-40:], c.v[0][-40:] = bad, bad
    again(c)
    c.k[0], c.v[0], c.lens[0] = c.k[0][:-40], c.v[0][:-40], lens[0] - 40
    c.len = torch.tensor(c.lens).cuda()
    hold(c, c.run())


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_windows_past_every_length(kh, window):
    """A window as wide as its type is none, for rows before the cache's first position too."""
    c = Case(BF16, 512, 4, 64, 16, [120, 0, 60, 40], [100, 9, 60, 300])
    unpacked(c, 120, 704, True)
    d = Case(F32, 8, 2, 64, 16, [5, 1, 2, 1], [2, 4000, 700, 1300])
    for x, dt, most in ((c, 2, dict(max_rows=120, max_len=704)), (d, 0, dict(max_rows=1, max_len=4000))):
        want = x.run(**most)
        # the workspace's memory holds no earlier call's parts or positions
        need = x.cache._workspace(dt, sum(x.rows), len(x.rows), x.heads, most["max_rows"], most["max_len"], 1)
        torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda")
        got = x.run(window=window, **most)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        x.cache.status()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [64, 128])
def test_single_rows_of_many_sequences_in_parts(kh, dtype, dim):
    """More than 64 sequences, each cut in the same number of parts; all share their first pages."""
    n = 70
    c = Case(dtype, 3, 1, dim, 16, [1] * n, [16 + (b * 97) % 2990 for b in range(n)])
    c.table[1:, 0] = c.table[0, 0]
    for b in range(1, n):
        c.k[b][:16], c.v[b][:16] = c.k[0][:16], c.v[0][:16]
    assert c.cache._workspace(0 if dtype == F32 else 2, n, n, 3, 1, 3005, 1) > 0
    hold(c, c.run(max_rows=1, max_len=3005))
    hold(c, c.run(max_rows=1, max_len=3005, window=900, return_lse=False), window=900)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 64), (16, 4, 128), (6, 2, 256)])
def test_log_sums_of_one_position(kh, dtype, heads, kv, dim):
    """The log-sum-exp of one position is its score, held to the roundings that the method's own numbers have.

    A score sums, group by group, s q (B + c) over 32 elements (B = 16 in BF16, 0 in f32), and s, m against sums of q: f32 additions, each off by
    u / sqrt(3) of its partial sum in the root mean square, u = 2^-24.  A group's 32 additions have partial sums of at
    most P = |q (B + c)| (2-norm, signs being independent), so they are off by u sqrt(32 / 3) s P together; its share of
    the second sum, of sizes B s |Q| and |m Q|, is added by some 8 at most: u sqrt(8 / 3) of those; the groups'
    sums are added once each, to a total within their 2-norm, and the score is scaled and turned to natural logarithms by
    four more roundings of itself."""
    n, u, bias = 300, 2.0 ** -24, 16 if dtype == BF16 else 0
    c = Case(dtype, heads, kv, dim, 16, [1] * n, [1] * n)
    _, lse = c.run(max_rows=1, max_len=1)
    q, k = c.q.double().numpy(), np.stack([x[0].float().numpy() for x in c.k])  # [n, heads, dim], [n, kv, dim]
    kc, ks, km = (np.repeat(x, heads // kv, 1).reshape(n, heads, dim // 32, 32) for x in quantize(k))
    q, s, m = q.reshape(n, heads, -1, 32), ks[..., 0], km[..., 0]
    want = ((q * (ks * kc + km)).sum((-2, -1))) * dim ** -0.5
    p, total = s * np.sqrt((q * q * (bias + kc) ** 2).sum(-1)), np.abs(q.sum(-1))
    each = 32 / 3 * p ** 2 + 8 / 3 * ((bias * s * total) ** 2 + (m * total) ** 2) + p ** 2 / 3
    bound = u * np.sqrt(each.sum(-1) / dim + 4 * want ** 2)
    off = lse.double().cpu().numpy() - want
    ratio = np.sqrt((off ** 2).mean() / (bound ** 2).mean())
    print(f"root mean square of the errors / of their bounds {ratio:.3f}")
    assert ratio <= 1


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
    torch.cuda.empty_cache()
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
    del q, out
    torch.cuda.empty_cache()

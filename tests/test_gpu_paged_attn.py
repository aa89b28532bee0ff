"""GPU: attention over the paged 4-bit cache against softmax attention in 64 bits over the values that the
cache stands for.  The tolerances are those of paged_ref.attention, derived there from the method's roundings."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, attention, keys, offsets

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


class Case:
    """Sequences with `rows` new rows and `lens` cached positions, filled from the host's rows."""

    def __init__(self, dtype, heads, kv, dim, page, rows, lens, seed=0, qscale=1.0):
        from klearu_amd import paged
        rng = np.random.default_rng(seed + heads * dim + page)
        self.dtype, self.heads, self.kv, self.dim, self.rows, self.lens = dtype, heads, kv, dim, rows, lens
        pg = Pages(lens, page, seed=seed)
        self.cache = paged.PagedKv(kv, dim, pg.pages, page_size=page)
        self.k = [torch.from_numpy(keys(rng, n, kv, dim)).to(dtype) for n in lens]
        self.v = [torch.from_numpy(keys(rng, n, kv, dim)).to(dtype) for n in lens]
        self.off, self.len, self.table = offsets(rows).cuda(), torch.tensor(lens, dtype=torch.int64).cuda(), pg.table.cuda()
        zero = torch.zeros(len(lens), dtype=torch.int64).cuda()
        if sum(lens):
            self.cache.append(torch.cat(self.k).cuda(), torch.cat(self.v).cuda(), offsets(lens).cuda(), zero, self.table)
        self.fine = False  # whether BF16 rows hold their weights in two terms
        self.many = False  # whether the call takes tiles of many rows
        self.q = torch.from_numpy((rng.normal(0, qscale, (sum(rows), heads, dim))).astype(np.float32)).to(dtype)

    def run(self, **kw):
        kw.setdefault("return_lse", True)
        n = max(1, -(-sum(self.rows) // len(self.rows)))
        self.many = self.dtype == BF16 and min(kw.get("max_rows", n), sum(self.rows)) * self.heads // self.kv >= 64
        return self.cache.attention(self.q.cuda(), self.off, self.len, self.table, **kw)

    def check(self, got, causal=True, window=0, scale=None, on=None):
        out, lse = (None if x is None else x.double().cpu().numpy() for x in ((got, None) if torch.is_tensor(got) else got))
        at, worst = 0, 0.0
        for n, length, k, v in zip(self.rows, self.lens, self.k, self.v):
            if n == 0:
                continue
            q = self.q[at:at + n].double().numpy()
            first = max(0, n - length)  # rows before the cache's first position see nothing
            keep = slice(at + first, at + n)
            assert causal or not first
            assert (out[at:at + first] == 0).all() and (lse is None or (lse[at:at + first] == -np.inf).all())
            if length:
                o, l, to, tl = attention(q[first:], k.float().numpy(), v.float().numpy(),
                                         self.dim ** -0.5 if scale is None else scale, causal, window, self.dtype == BF16, self.many, self.fine)
                if on is not None:
                    off = ~on[keep]
                    o[off], l[off], to[off], tl[off] = 0, -np.inf, 0, 0
                assert (np.isnan(out[keep]) == np.isnan(o)).all()
                fine = ~np.isnan(o)
                d = np.abs(out[keep] - o)
                assert (d[fine] <= to[fine]).all(), float(np.nanmax(np.where(fine, d - to, 0)))
                worst = max(worst, float(np.max(np.where(fine & (to > 0), d / np.where(to > 0, to, 1), 0), initial=0)))
                some = np.isfinite(l)
                if lse is None:
                    at += n
                    continue
                assert (lse[keep][~some & ~np.isnan(l)] == -np.inf).all()
                assert (np.abs(lse[keep][some] - l[some]) <= tl[some]).all()
            at += n
        print(f"worst error / tolerance {worst:.3f}")
        self.cache.status()


SHAPES = [(1, 1, 64), (4, 4, 128), (8, 2, 64), (8, 1, 128), (16, 2, 256), (6, 2, 128), (3, 1, 256), (40, 2, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
def test_single_rows(kh, dtype, heads, kv, dim, page):
    """One row per sequence, lengths around every border, an empty one among them."""
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]
    c = Case(dtype, heads, kv, dim, page, [1] * len(lens), lens)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (8, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 40), (False, 0)])
def test_many_rows(kh, dtype, heads, kv, dim, page, causal, window):
    """Prompts, chunks over what is cached, one row, none."""
    rows, lens = [70, 0, 1, 33, 5], [70, 40, 90, 133, 200]
    c = Case(dtype, heads, kv, dim, page, rows, lens)
    c.check(c.run(causal=causal, window=window), causal, window)
    c.check(c.run(causal=causal, window=window, return_lse=False), causal, window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim,length", [(4, 4, 128, 5000), (8, 1, 64, 9001), (2, 1, 256, 4097)])
@pytest.mark.parametrize("window", [0, 1000])
def test_long(kh, dtype, heads, kv, dim, length, window):
    """Split along the positions and joined."""
    c = Case(dtype, heads, kv, dim, 64, [1], [length])
    c.check(c.run(window=window), window=window)
    if not window:
        c = Case(dtype, heads, kv, dim, 16, [3, 1], [length, 77])
        c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_prompt_of_many_tiles(kh, dtype):
    c = Case(dtype, 8, 2, 128, 64, [530, 259], [530, 700])
    c.check(c.run(max_rows=530, max_len=700))
    c.check(c.run(window=100), window=100)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_before_the_cache(kh, dtype):
    """More new rows than positions: the first of them see nothing."""
    c = Case(dtype, 4, 2, 128, 16, [40, 3, 20], [10, 0, 20])
    c.check(c.run())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv", [(8, 8), (8, 2)])
@pytest.mark.parametrize("rows,lens", [([1, 1], [900, 65]), ([20, 1, 7], [20, 50, 700])])
def test_selected_heads(kh, dtype, heads, kv, rows, lens):
    """Lists as the head predictor gives them; ids outside and repeated ones; an empty list."""
    c = Case(dtype, heads, kv, 128, 64, rows, lens)
    n = sum(rows)
    rng = np.random.default_rng(1)
    sel = np.stack([rng.permutation(heads)[:3] for _ in range(n)]).astype(np.int32)
    sel = np.concatenate([sel, np.tile(np.int32([[-1, heads, 70000]]), (n, 1)), sel[:, :1]], 1)
    sel[0] = -5
    on = np.zeros((n, heads), bool)
    for t in range(n):
        on[t, [h for h in sel[t] if 0 <= h < heads]] = True
    c.check(c.run(heads=torch.from_numpy(sel).cuda()), on=on)
    none = c.run(heads=torch.zeros(n, 0, dtype=torch.int32).cuda())
    assert (none[0] == 0).all() and (none[1] == -np.inf).all()


def test_predictors_lists(kh, orc):
    """The head predictor's own selection drives it, as in the framework's decode step."""
    from klearu_amd.dejavu import ORDER_ASCENDING, SparsityPredictor
    rng = np.random.default_rng(6)
    hidden, heads, k = 256, 8, 3
    p = SparsityPredictor(rng.normal(0, .1, (16, hidden)).astype(np.float32), np.zeros(16, np.float32),
                          rng.normal(0, .3, (heads, 16)).astype(np.float32), np.zeros(heads, np.float32))
    ids = p.select_top_k(torch.randn(3, hidden, device="cuda"), k, ORDER_ASCENDING)
    c = Case(F32, heads, heads, 64, 32, [1, 1, 1], [40, 100, 7])
    on = np.zeros((3, heads), bool)
    np.put_along_axis(on, ids.cpu().numpy().astype(np.int64), True, 1)
    c.check(c.run(heads=ids), on=on)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_peaks_and_scales(kh, dtype):
    """Scores far apart, one position that takes all, tiny and large scales."""
    for qs, scale in ((30.0, None), (1.0, 1e-4), (1.0, 3.0), (0.0, None)):
        c = Case(dtype, 4, 2, 64, 16, [1, 9], [333, 50], qscale=qs)
        c.check(c.run(scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows", [[1, 1], [40, 25]])
@pytest.mark.parametrize("where", ["k", "v"])
def test_values_that_are_not_finite(kh, dtype, rows, where):
    """NaN and infinities: rows that see the position get NaN (of a value's group alone), rows that do not see it,
    behind the causal border or the window, are as if it were not there; nor do recycled pages leave a trace."""
    rng = np.random.default_rng(7)
    lens = [200, 150]
    for bad in (np.nan, np.inf, -np.inf):
        c = Case(dtype, 4, 2, 64, 16, rows, lens)
        zero = torch.zeros(2, dtype=torch.int64).cuda()
        x = c.k if where == "k" else c.v
        # one in the middle of sequence 0's new rows or near its end, one that a window leaves behind
        x[0][lens[0] - (rows[0] + 1) // 2, 1, 40] = bad
        x[1][3, 0, 0] = bad
        c.cache.append(torch.cat(c.k).cuda(), torch.cat(c.v).cuda(), offsets(lens).cuda(), zero, c.table)
        c.check(c.run(window=64), window=64)
        c.check(c.run())


def test_recycled_pages(kh):
    """Pages full of NaN groups, handed to a shorter sequence: what lies behind its length does not count."""
    from klearu_amd import paged
    cache = paged.PagedKv(2, 64, 3, page_size=64)
    t = torch.tensor([[1, 2]], dtype=torch.int32).cuda()
    nan = torch.full((128, 2, 64), float("nan"), device="cuda")
    one, z = torch.zeros(1, dtype=torch.int64).cuda(), offsets([128]).cuda()
    cache.append(nan, nan, z, one, t)
    rng = np.random.default_rng(1)
    k, v = (torch.from_numpy(keys(rng, 70, 2, 64)) for _ in range(2))
    cache.append(k.cuda(), v.cuda(), offsets([70]).cuda(), one, t)
    q = torch.from_numpy(rng.normal(0, 1, (1, 4, 64)).astype(np.float32))
    for dtype in (F32, BF16):
        got = cache.attention(q.to(dtype).cuda(), offsets([1]).cuda(), torch.tensor([70]).cuda(), t)
        o, _, to, _ = attention(q.to(dtype).double().numpy(), k.numpy(), v.numpy(), 0.125, bf16=dtype == BF16)
        assert (np.abs(got.double().cpu().numpy() - o) <= to).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides(kh, dtype, shift):
    """Queries inside projection rows, heads-first outputs, unaligned starts: the packed call's bits, and
    nothing else written."""
    for rows, lens in (([1, 1, 1], [50, 700, 3]), ([30, 80], [30, 100])):
        c = Case(dtype, 8, 2, 128, 32, rows, lens)
        n = sum(rows)
        want = c.run()
        buf = torch.full((n * 12 * 128 + shift,), 9.0, dtype=dtype, device="cuda")[shift:].view(n, 12, 128)
        buf[:, 2:10] = c.q.cuda()
        flat = torch.full((8 * (n + 1) * 128 + shift,), 4.0, dtype=dtype, device="cuda")[shift:].view(8, n + 1, 128)
        out = flat[:, :n].transpose(0, 1)
        got = c.cache.attention(buf[:, 2:10], c.off, c.len, c.table, out=out, return_lse=True)
        assert got[0] is out and torch.equal(out, want[0]) and torch.equal(got[1], want[1])
        assert (flat[:, n] == 4).all()
        # without the log-sum-exp tiles of many rows hold their keys in one BF16 term
        alone = c.cache.attention(c.q.cuda(), c.off, c.len, c.table)
        c.check(alone)
        wide = torch.full((n, 12, 128), 4.0, dtype=dtype, device="cuda")
        c.cache.attention(c.q.cuda(), c.off, c.len, c.table, out=wide[:, :8])
        assert torch.equal(wide[:, :8], alone) and (wide[:, 8:] == 4).all()
        # a table's columns inside a wider one
        big = torch.full((len(rows), c.table.shape[1] + 3), -9, dtype=torch.int32, device="cuda")
        big[:, 2:-1] = c.table
        assert torch.equal(c.cache.attention(c.q.cuda(), c.off, c.len, big[:, 2:-1]), alone)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_guesses_and_padding(kh, dtype):
    """Wrong guesses of rows and lengths give right results; padding rows keep what they held."""
    c = Case(dtype, 8, 2, 64, 16, [1, 90, 0, 17], [2000, 90, 5, 300])
    for r, l in ((1, 1), (1, 10 ** 6), (90, 2000), (10 ** 6, 1), (0, 0)):
        c.check(c.run(max_rows=r, max_len=l))
    n = sum(c.rows)
    for split in (1, 2000):
        q = torch.cat([c.q[:2] * 0 + 3, c.q, c.q[:5]]).cuda()
        out = torch.full_like(q, 6.0)
        c.cache.attention(q, c.off + 2, c.len, c.table, out=out, max_len=split, max_rows=1)
        c.check((out[2:n + 2], c.run()[1]))
        assert (out[:2] == 6).all() and (out[n + 2:] == 6).all()


def test_no_rows(kh):
    c = Case(BF16, 2, 1, 64, 16, [0, 0], [5, 0])
    assert c.run()[0].shape == (0, 2, 64)
    e = torch.zeros(0, dtype=torch.int64).cuda()
    out = torch.full((3, 2, 64), 2.0, device="cuda")
    c.cache.attention(out.clone(), torch.zeros(1, dtype=torch.int64).cuda(), e, torch.zeros(0, 1, dtype=torch.int32).cuda(), out=out)
    assert (out == 2).all()


def test_bad_pages_are_reported(kh):
    """Pages outside the pool and lengths past the table: nothing there is read, the rest counts, and status says so;
    entries behind the length or before the window are not looked at."""
    from klearu_amd import KlearuError
    for page in (16, 64):
        c = Case(F32, 2, 1, 64, page, [1], [100])
        want = c.run()
        c.cache.status()
        bad = c.table.clone()
        bad[0, 0] = 10 ** 6
        got = c.cache.attention(c.q.cuda(), c.off, c.len, bad)
        with pytest.raises(KlearuError, match="page id"):
            c.cache.status()
        # as if the page's positions were not there
        o, _, to, _ = attention(c.q.double().numpy(), c.k[0][page:].float().numpy(), c.v[0][page:].float().numpy(), 0.125,
                                bf16=False)
        assert (np.abs(got.double().cpu().numpy() - o) <= to).all()
        # with a window, freed pages may be anything
        w = 100 - page
        c.check((c.cache.attention(c.q.cuda(), c.off, c.len, bad, window=w, return_lse=True)), window=w)
        c.cache.status()
        got = c.cache.attention(c.q.cuda(), c.off, torch.tensor([10 ** 9]).cuda(), c.table)
        with pytest.raises(KlearuError, match="page"):
            c.cache.status()
        got = c.cache.attention(c.q.cuda(), c.off, torch.tensor([-4]).cuda(), c.table)
        assert (got == 0).all()
        with pytest.raises(KlearuError, match="page table"):
            c.cache.status()
        assert torch.equal(c.run()[0], want[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_call_same_bits(kh, dtype):
    c = Case(dtype, 8, 2, 128, 64, [1, 50], [3000, 800])
    a = c.run()
    for _ in range(3):
        b = c.run()
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_streams_at_once(kh):
    """Two calls over one cache on two streams, each with its own workspace."""
    c, d = Case(BF16, 8, 2, 128, 64, [1], [5000]), Case(BF16, 8, 2, 128, 64, [2], [3000], seed=5)
    a, b = c.run(), d.run()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    qs = [x.q.cuda() for x in (c, d)]
    torch.cuda.synchronize()
    got = []
    for _ in range(10):
        got.append((c.cache.attention(qs[0], c.off, c.len, c.table, stream=s),
                    d.cache.attention(qs[1], d.off, d.len, d.table, stream=t)))
    torch.cuda.synchronize()
    for x, y in got:
        assert torch.equal(x, a[0]) and torch.equal(y, b[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decode_steps_in_a_graph(kh, dtype):
    """The run of them as a model's step has it: rotate the queries, append keys and values with their
    rotation, attend, lengths advanced; captured once and replayed, eager work between, against eager steps
    over a second cache and against 64 bits at the end."""
    from klearu_amd import paged
    rng = np.random.default_rng(11)
    heads, kv, dim, page, b, steps = 8, 2, 128, 16, 3, 40
    lens = [0, 700, 33]
    pg = Pages([n + steps for n in lens], page)
    rope = paged.Rope(dim, 4096)
    caches = [paged.PagedKv(kv, dim, pg.pages, page_size=page) for _ in range(2)]
    tb, off = pg.table.cuda(), offsets([1] * b).cuda()
    pre_k, pre_v = ([torch.from_numpy(keys(rng, n, kv, dim)).to(dtype) for n in lens] for _ in range(2))
    zero = torch.zeros(b, dtype=torch.int64).cuda()
    for c in caches:
        c.append(torch.cat(pre_k).cuda(), torch.cat(pre_v).cuda(), offsets(lens).cuda(), zero, tb, rope=rope)
    qkv = torch.zeros(b, heads + 2 * kv, dim, dtype=dtype, device="cuda")
    start = torch.tensor(lens).cuda()
    at = [start.clone(), start.clone()]
    out = torch.zeros(b, heads, dim, dtype=dtype, device="cuda")

    def step(c, pos):
        q = rope.apply(qkv[:, :heads], pos)
        c.append(qkv[:, heads:heads + kv], qkv[:, heads + kv:], off, pos, tb, rope=rope)
        pos += 1
        return c.attention(q, off, pos, tb, max_rows=1, max_len=1000)

    step(caches[1], at[1].clone())  # warm, on places that are written again
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out.copy_(step(caches[0], at[0]))
    rows = []
    for i in range(steps):
        new = torch.from_numpy(keys(rng, b, heads + 2 * kv, dim)).to(dtype)
        qkv.copy_(new)
        rows.append(new)
        g.replay()
        want = step(caches[1], at[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
    for c in caches:
        c.status()
    rope.status()
    pos = torch.tensor([n + steps - 1 for n in lens]).cuda()
    q = rope.apply(qkv[:, :heads], pos).double().cpu().numpy()
    rot = paged.Rope(dim, 4096)
    for s in range(b):
        n = lens[s] + steps
        k = torch.cat([pre_k[s]] + [r[s:s + 1, heads:heads + kv] for r in rows])
        v = torch.cat([pre_v[s]] + [r[s:s + 1, heads + kv:] for r in rows])
        k = rot.apply(k.float().cuda(), torch.arange(n).cuda()).cpu().numpy()
        o, _, to, _ = attention(q[s:s + 1], k, v.float().numpy(), dim ** -0.5, bf16=dtype == BF16)
        assert (np.abs(out[s:s + 1].double().cpu().numpy() - o) <= to).all()


def test_two_graphs_of_one_stream(kh):
    """Two captured calls replayed at once on two streams: workspaces of their own."""
    c, d = Case(BF16, 8, 2, 128, 64, [1], [5000]), Case(BF16, 8, 2, 128, 64, [1], [4000], seed=5)
    qs = [x.q.cuda() for x in (c, d)]
    want = [x.run()[0] for x in (c, d)]
    outs = [torch.zeros_like(w) for w in want]
    graphs = []
    torch.cuda.synchronize()
    for x, q, o in zip((c, d), qs, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.cache.attention(q, x.off, x.len, x.table, out=o)
        graphs.append(g)
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(8):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for g, st in zip(graphs, s):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


# Row tiles enough that the positions are unpacked ahead of them (BF16)
AHEAD = [(32, 2, 64, [60, 40], [60, 300]), (64, 4, 128, [40, 0, 70], [40, 9, 450]), (32, 2, 256, [50, 33], [180, 33])]


@pytest.mark.parametrize("heads,kv,dim,rows,lens", AHEAD)
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 70), (False, 0)])
def test_unpacked_ahead(kh, heads, kv, dim, rows, lens, page, causal, window):
    c = Case(BF16, heads, kv, dim, page, rows, lens)
    for lse in (True, False):
        c.check(c.run(causal=causal, window=window, max_rows=max(rows), max_len=max(lens), return_lse=lse), causal, window)
    # a sequence longer than the caller says, and lengths far shorter
    for most in (max(lens) - 64, 64, 10 ** 5):
        for lse in (True, False):
            c.check(c.run(causal=causal, window=window, max_rows=max(rows), max_len=most, return_lse=lse), causal, window)


@pytest.mark.parametrize("heads,kv,dim,rows,lens", AHEAD)
def test_unpacked_ahead_values_that_are_not_finite(kh, heads, kv, dim, rows, lens):
    c = Case(BF16, heads, kv, dim, 16, rows, lens)
    for b, n in enumerate(lens):
        if n > 20:
            c.v[b][n - 3, kv - 1, dim - 1] = float("nan")  # the last rows see it, and one group of them turns
            c.v[b][n - rows[b] // 2, 0, 33] = float("inf")
            c.k[b][n - rows[b] // 3, kv // 2, 5] = float("nan")
    c.cache.append(torch.cat(c.k).cuda(), torch.cat(c.v).cuda(), offsets(lens).cuda(),
                   torch.zeros(len(lens), dtype=torch.int64).cuda(), c.table)
    for lse in (True, False):
        c.check(c.run(max_rows=max(rows), max_len=max(lens), return_lse=lse))
        c.check(c.run(max_rows=max(rows), max_len=max(lens), window=30, return_lse=lse), window=30)


@pytest.mark.parametrize("heads,kv,dim,rows,lens", AHEAD)
def test_unpacked_ahead_pages_and_heads(kh, heads, kv, dim, rows, lens):
    """A page that is not there leaves the rest; freed pages before a window are not looked at; listed heads alone."""
    from klearu_amd import KlearuError
    c = Case(BF16, heads, kv, dim, 16, rows, lens)
    c.many = True
    q, most = c.q.cuda(), dict(max_rows=max(rows), max_len=max(lens))
    last = len(lens) - 1
    bad = c.table.clone()
    bad[last, 0] = -7
    got = c.cache.attention(q, c.off, c.len, bad, **most)
    with pytest.raises(KlearuError, match="page id"):
        c.cache.status()
    at, n, length = sum(rows[:last]), rows[last], lens[last]
    late = [i for i in range(n) if length - n + i >= 16]
    qs = c.q[[at + i for i in late]].double().numpy()
    for i, row in list(zip(late, qs))[:: max(1, len(late) // 5)]:
        k, v = (x[last][16:length - n + i + 1].float().numpy() for x in (c.k, c.v))
        o, _, to, _ = attention(row[None], k, v, dim ** -0.5, many=True)
        assert (np.abs(got[at + i].double().cpu().numpy() - o[0]) <= to[0]).all()
    if length - n - 20 >= 16:
        c.check(c.cache.attention(q, c.off, c.len, bad, window=20, return_lse=True, **most), window=20)
    rng = np.random.default_rng(2)
    sel = np.stack([rng.permutation(heads)[:5] for _ in range(sum(rows))]).astype(np.int32)
    on = np.zeros((sum(rows), heads), bool)
    np.put_along_axis(on, sel.astype(np.int64), True, 1)
    c.check(c.run(heads=torch.from_numpy(sel).cuda(), **most), on=on)


def test_unpacked_ahead_in_a_graph(kh):
    """A prompt's attention captured and replayed, eager calls between: no workspace is shared."""
    c = Case(BF16, 32, 2, 128, 64, [70, 30], [70, 200])
    q, out = c.q.cuda(), torch.zeros_like(c.q, device="cuda")
    kw = dict(max_rows=70, max_len=200)
    want = c.cache.attention(q, c.off, c.len, c.table, **kw)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.cache.attention(q, c.off, c.len, c.table, out=out, **kw)
    for _ in range(4):
        out.zero_()
        g.replay()
        other = c.cache.attention(q * 0.5, c.off, c.len, c.table, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and not torch.equal(other, want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim,lens", [
    (8, 2, 64, [4000, 1, 700, 0, 33, 1300, 64, 2600]), (4, 1, 128, [3000, 3000]), (2, 2, 256, [1, 5000, 0, 1]),
    (4, 4, 64, [1 + 61 * i for i in range(40)])])
@pytest.mark.parametrize("window", [0, 500])
def test_ragged_lengths_share_the_parts(kh, dtype, heads, kv, dim, lens, window):
    """Single rows whose parts are dealt out by length, one sequence without a row, two rows in another; a guess of
    the longest that is far too large."""
    rows = [1] * len(lens)
    rows[-1] = 2 if lens[-1] >= 2 else 1
    rows[len(lens) // 2] = 0 if len(lens) > 2 else 1
    c = Case(dtype, heads, kv, dim, 32, rows, lens)
    for most in (max(lens), 10 ** 6):
        got = c.run(window=window, max_rows=1, max_len=most)
        c.check(got, window=window)
        again = c.run(window=window, max_rows=1, max_len=most)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


# Row tiles enough, or said to go far enough, for the tiles of many rows (BF16): the guess of the longest length
# decides whether they are split along the positions and whether these are unpacked ahead.
TILES = [(64, 4, 64, [70, 0, 50, 1], [70, 40, 333, 20]), (64, 4, 128, [160, 30, 0, 95], [160, 30, 9, 450]),
         (32, 2, 256, [150, 0, 90, 100], [180, 5, 90, 333])]


@pytest.mark.parametrize("heads,kv,dim,rows,lens", TILES)
@pytest.mark.parametrize("guess", [500, 1999, 10 ** 5])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 1), (True, 70), (False, 0)])
@pytest.mark.parametrize("lse", [True, False])
def test_tiles_of_many_rows(kh, heads, kv, dim, rows, lens, guess, causal, window, lse):
    c = Case(BF16, heads, kv, dim, 16 if causal else 64, rows, lens)
    c.check(c.run(causal=causal, window=window, max_rows=max(rows), max_len=guess, return_lse=lse), causal, window)


@pytest.mark.parametrize("heads,kv,dim,rows,lens", TILES)
@pytest.mark.parametrize("guess", [500, 1999, 10 ** 5])
def test_tiles_of_many_rows_not_finite_lists_pages(kh, heads, kv, dim, rows, lens, guess):
    """Groups that stand for NaN reach the rows that see them alone; unlisted heads; a page that is not there
    before the window."""
    c = Case(BF16, heads, kv, dim, 16, rows, lens)
    last = len(lens) - 1
    c.v[2 if lens[2] > 50 else last][lens[2] - 3 if lens[2] > 50 else lens[last] - 3, kv - 1, dim - 1] = float("nan")
    c.k[0][lens[0] - 10, 0, 5] = float("inf")
    c.cache.append(torch.cat(c.k).cuda(), torch.cat(c.v).cuda(), offsets(lens).cuda(),
                   torch.zeros(len(lens), dtype=torch.int64).cuda(), c.table)
    most = dict(max_rows=max(rows), max_len=guess)
    for lse in (True, False):
        c.check(c.run(return_lse=lse, **most))
    rng = np.random.default_rng(2)
    sel = np.stack([rng.permutation(heads)[:5] for _ in range(sum(rows))]).astype(np.int32)
    on = np.zeros((sum(rows), heads), bool)
    np.put_along_axis(on, sel.astype(np.int64), True, 1)
    c.check(c.run(heads=torch.from_numpy(sel).cuda(), **most), on=on)
    if lens[last] - rows[last] - 20 >= 16:
        c.table[last, 0] = -7
        c.check(c.run(window=20, **most), window=20)


@pytest.mark.parametrize("guess", [1999, 10 ** 5])
def test_tiles_of_many_rows_in_a_graph(kh, guess):
    c = Case(BF16, *TILES[1][:3], 64, *TILES[1][3:])
    q, out = c.q.cuda(), torch.zeros_like(c.q, device="cuda")
    kw = dict(max_rows=160, max_len=guess)
    want = c.cache.attention(q, c.off, c.len, c.table, **kw)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        c.cache.attention(q, c.off, c.len, c.table, out=out, **kw)
    for _ in range(4):
        out.zero_()
        g.replay()
        other = c.cache.attention(q * 0.5, c.off, c.len, c.table, **kw)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and not torch.equal(other, want)


@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 128), (8, 2, 64), (6, 2, 256)])
@pytest.mark.parametrize("rows,lens,window", [([1] * 6, [1, 7, 20, 33, 150, 512], 0), ([9, 1, 4], [9, 40, 333], 0),
                                              ([1, 3, 1], [2000, 900, 31], 24)])
def test_few_positions(kh, heads, kv, dim, rows, lens, window):
    """BF16 rows of 512 positions or fewer, by their lengths or a window: weights to 2^-16."""
    c = Case(BF16, heads, kv, dim, 32, rows, lens)
    c.fine = True
    got = c.run(window=window, max_len=max(lens))
    c.many = False
    c.check(got, window=window)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("heads,kv,dim,lens", [(1, 1, 64, [40000, 25001]), (2, 1, 128, [30000, 1, 17])])
def test_most_parts_of_a_row(kh, dtype, heads, kv, dim, lens):
    """Few sequences of one kv head over long caches: as many parts as the join takes."""
    c = Case(dtype, heads, kv, dim, 256, [1] * len(lens), lens)
    for most in (max(lens), 2 ** 31):
        c.check(c.run(max_len=most))
        c.check(c.run(max_len=most, return_lse=False))


@pytest.mark.parametrize("rows,guess", [(5, 40), (33, 1999)])
def test_many_rows_of_many_sequences(kh, rows, guess):
    """More than 64 sequences in tiles of many rows, some without rows."""
    n = [0 if i % 7 == 3 else 1 + i % rows for i in range(70)]
    c = Case(BF16, 64, 4, 64, 16, n, [r + i % 9 for i, r in enumerate(n)])
    for lse in (True, False):
        c.check(c.run(max_rows=rows, max_len=guess, return_lse=lse))

"""GPU: attention weights of cached positions against 64 bits.

A weight is exp(x), x = scale q . k - lse.  x is off by the f32 sums of the score (at most dim + 32 additions of
magnitudes B = scale sum |q| (15 s + |m|)), by the conversion of lse to powers of two (2 * 2^-24 |lse|) and by a last
fused addition (2^-24 |x|), by d in all: exp(x + d) - exp(x) = exp(x) (exp(d) - 1), so the weight by that (scores of 1e8 and
more have no f32 digits behind the point: d passes 1, and the tolerance says nothing there); the exponential by 2^-22 of itself and, through x log2 e, 2^-23 |x|.  Sums of R weights take at most
R / 4 + 64 additions in a row, each off by 2^-24 of the sum, and acc itself is rounded once."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, bf16_values, keys, offsets, quantize, seen, values

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(q, lse, kraw, scale, causal, window):
    """One sequence: q [n, heads, dim] f64, lse [n, heads] f32, kraw [length, kv, dim] -> (sums, tolerance) [kv, length]."""
    n, heads, dim = q.shape
    length, kv = kraw.shape[:2]
    _, s, m = quantize(kraw)
    k, ok = values(kraw), seen(n, length, causal, window)
    out, tol = np.zeros((kv, length)), np.zeros((kv, length))
    for h in range(heads):
        g, l = h * kv // heads, lse[:, h].astype(np.float64)[:, None]
        on = ok & ~np.isinf(l)
        with np.errstate(all="ignore"):
            x = np.where(on, q[:, h] @ k[:, g].T * scale - l, -np.inf)
            p = np.exp(x)
            big = scale * (np.abs(q[:, h]) @ (15 * s[:, g] + np.abs(m[:, g])).T)
            err = np.where(on, ((dim + 32) * big + 2 * np.abs(l) + 3 * np.abs(x) + 4) * U, 0.0)
        out[g] += np.where(on, p, 0.0).sum(0)
        err = np.nan_to_num(err)
        tol[g] += np.where(err > 1, np.inf, np.where(on, p, 0.0) * np.expm1(np.minimum(err, 1.0))).sum(0)
    return out, tol + (n * heads / kv / 4 + 64) * U * out


class Call:
    """A call's inputs from sizes: sequences of rows and lengths, keys, queries and log-sum-exps in 64 bits."""

    def __init__(self, heads, kv, dim, rows, lens, page=16, dtype=torch.bfloat16, causal=True, window=0, seed=0, spare=1, k=None):
        from klearu_amd import paged
        rng = np.random.default_rng(seed + dim + sum(lens))
        self.rows, self.lens, self.causal, self.window, self.scale = rows, lens, causal, window, dim ** -0.5
        self.pages = Pages(lens, page, spare=spare)
        self.cache = paged.PagedKv(kv, dim, self.pages.pages, page_size=page)
        self.k = [keys(rng, n, kv, dim) for n in lens] if k is None else k
        self.table = self.pages.table.cuda()
        self.off, self.len = offsets(rows).cuda(), torch.tensor(lens).cuda()
        flat = torch.from_numpy(np.concatenate(self.k)).cuda()
        self.cache.append(flat, flat, offsets(lens).cuda(), torch.zeros_like(self.len), self.table)
        self.q = torch.from_numpy(rng.normal(0, 1.2, (sum(rows), heads, dim)).astype(np.float32)).to(dtype)
        self.lse = np.full((sum(rows), heads), -np.inf, np.float32)
        at = 0
        for n, length, kr in zip(rows, lens, self.k):
            x, ok = self.q[at:at + n].double().numpy(), seen(n, length, causal, window)
            for h in range(heads):
                y = np.where(ok, x[:, h] @ values(kr)[:, h * kv // heads].T * self.scale, -np.inf)
                top = y.max(-1, initial=-np.inf)
                some = np.isfinite(top)
                with np.errstate(all="ignore"):
                    self.lse[at:at + n, h] = np.where(some, top + np.log(np.exp(y - np.where(some, top, 0)[:, None]).sum(-1)), top)
            at += n
        self.acc = torch.from_numpy(rng.exponential(1, (len(lens), kv, self.table.shape[1] * page)).astype(np.float32))

    def run(self, q=None, lse=None, acc=None, **kw):
        args = dict(causal=self.causal, window=self.window, max_rows=max(self.rows), max_len=max(self.lens))
        args.update(kw)
        return self.cache.attention_weights((self.q if q is None else q).cuda(), torch.as_tensor(self.lse if lse is None else lse).cuda(),
                                            self.off, self.len, self.table, self.acc.cuda() if acc is None else acc, **args)

    def check(self, got, q=None, lse=None):
        q, lse, at = self.q if q is None else q, self.lse if lse is None else lse, 0
        got = got.double().cpu().numpy()
        for b, (n, length, kr) in enumerate(zip(self.rows, self.lens, self.k)):
            want, tol = reference(q[at:at + n].double().numpy(), lse[at:at + n], kr, self.scale, self.causal, self.window)
            old = self.acc[b].double().numpy()
            total = old[:, :length] + want
            d = np.abs(got[b, :, :length] - total)
            nan = np.isnan(total)
            assert np.array_equal(nan, np.isnan(got[b, :, :length])), b
            lim = tol + 2 * U * np.abs(total)
            assert (d <= lim)[~nan].all(), (b, float((d - lim)[~nan].max()))
            assert np.array_equal(got[b, :, length:], old[:, length:]), b  # nothing behind the sequence
            at += n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 64, 16), (8, 2, 128, 64), (2, 2, 256, 32), (6, 1, 64, 256), (32, 2, 128, 16)])
@pytest.mark.parametrize("rows,lens", [([1], [1]), ([1, 1, 1, 1], [15, 16, 700, 64]), ([5, 1, 0, 37], [5, 129, 40, 300])])
def test_weights(kh, dtype, heads, kv, dim, page, rows, lens):
    c = Call(heads, kv, dim, rows, lens, page, dtype)
    c.check(c.run())
    c.cache.status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 64), (4, 1, 128), (2, 1, 256)])
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 17), (True, 100), (True, 2 ** 40)])
def test_masks(kh, dtype, heads, kv, dim, causal, window):
    c = Call(heads, kv, dim, [70, 1, 130], [70, 333, 290], 32, dtype, causal, window if window < 2 ** 31 else 0)
    c.check(c.run(window=window))
    c.cache.status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,rows,lens,window", [
    (8, 2, 128, [700], [700], 0), (8, 2, 64, [513, 260], [1500, 260], 0), (4, 2, 256, [300, 1], [1111, 2000], 0),
    (4, 4, 128, [400, 333], [400, 900], 150), (16, 1, 128, [129], [2100], 0)])
def test_many_rows(kh, dtype, heads, kv, dim, rows, lens, window):
    c = Call(heads, kv, dim, rows, lens, 64, dtype, True, window)
    c.check(c.run())
    c.cache.status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,lens", [([9, 1], [4, 1]), ([300], [40]), ([3, 2], [0, 0])])
def test_rows_before_the_cache(kh, dtype, rows, lens):
    """More rows than positions: the first of them see nothing."""
    for causal in (True, False):
        c = Call(4, 2, 64, rows, lens, 16, dtype, causal)
        c.check(c.run(max_len=64))


@pytest.mark.parametrize("rows", [[1, 1], [200, 90]])
def test_log_sum_exps_that_are_not_finite(kh, rows):
    """Infinite ones add nothing, whatever the row holds; NaN makes the positions that the row sees NaN."""
    c = Call(4, 2, 128, rows, [300, 290])
    c.lse[0, 1], c.lse[-1, 2] = -np.inf, np.inf
    c.q[0, 1], c.q[-1, 2] = np.nan, np.inf
    clean = c.q.clone()
    clean[0, 1] = clean[-1, 2] = 0
    c.check(c.run(), q=clean)
    c.lse[-1, 0] = np.nan
    got = c.run().cpu()
    assert got[1, 0, :290].isnan().all() and not got[1, 1].isnan().any() and not got[0].isnan().any()
    assert not got[1, 0, 290:].isnan().any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [[1], [150]])
def test_keys_that_are_not_finite(kh, dtype, rows):
    """A position whose key has a NaN group gets NaN, no other one does."""
    c = Call(4, 2, 128, rows, [400], 32, dtype)
    lse = c.lse.copy()
    bad = Call(4, 2, 128, rows, [400], 32, dtype, k=[c.k[0].copy()])
    k = c.k[0].copy()
    k[5, 0, 3], k[211, 1, 127], k[399, 0, 64] = np.nan, np.inf, -np.inf
    flat = torch.from_numpy(k).cuda()
    bad.cache.append(flat, flat, offsets([400]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), bad.table)
    bad.k = [k]
    got = bad.run(lse=lse)
    bad.check(got, lse=lse)
    assert got.isnan().sum().item() == 3
    lse[:, :2] = -np.inf  # rows that add nothing add no NaN either
    got = bad.run(lse=lse)
    bad.check(got, lse=lse)
    assert not got[0, 0].isnan().any() and got[0, 1].isnan().sum().item() == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [[3], [150]])
@pytest.mark.parametrize("lo,hi", [(0, 0), (-3, 3), (-30, 30)])
def test_sizes_of_rows_and_keys(kh, dtype, rows, lo, hi):
    """Rows and keys of sizes that are powers of two apart, single large elements and zero rows, each position and row to
    its own tolerance (scales are chosen per position and row)."""
    rng = np.random.default_rng(hi)
    k = keys(rng, 400, 2, 128) * 2.0 ** rng.integers(lo, hi + 1, (400, 2, 1))
    k[7], k[300, 0, 5] = 0, 1000.0
    c = Call(4, 2, 128, rows, [400], 32, dtype, k=[k.astype(np.float32)])
    q = c.q.float() * torch.from_numpy(2.0 ** rng.integers(lo, hi + 1, c.q.shape[:2] + (1,))).float() * 2.0 ** -hi
    q[-1, 1], q[0, 3, 77] = 0, 8 * 2.0 ** -hi
    c.q = q.to(dtype)
    lse = np.zeros_like(c.lse)
    for h in range(4):  # a weight of at most 1 for each row
        x = np.where(seen(rows[0], 400, True, 0), c.q[:, h].double().numpy() @ values(c.k[0])[:, h // 2].T * c.scale, -np.inf)
        lse[:, h] = x.max(-1) + 1
    c.check(c.run(lse=lse), lse=lse)
    lse[lse > 1e4] = -np.inf  # without the rows whose scores have no digits left
    c.check(c.run(lse=lse), lse=lse)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [[3], [150]])
@pytest.mark.parametrize("power", [-80, 80, 90])
def test_large_scales(kh, dtype, rows, power):
    """Keys of 2^power and queries of 2^-power: ordinary scores of numbers whose scales are far from one."""
    rng = np.random.default_rng(power + 100)
    c = Call(4, 2, 128, rows, [300], 32, dtype, k=[(keys(rng, 300, 2, 128) * 2.0 ** power).astype(np.float32)])
    c.q = (c.q.double() * 2.0 ** -power).to(dtype)
    lse = np.zeros_like(c.lse)
    for h in range(4):
        x = np.where(seen(rows[0], 300, True, 0), c.q[:, h].double().numpy() @ values(c.k[0])[:, h // 2].T * c.scale, -np.inf)
        lse[:, h] = x.max(-1) + 1
    c.check(c.run(lse=lse), lse=lse)


@pytest.mark.parametrize("window", [0, 20])
def test_many_sequences(kh, window):
    """More sequences than a wave has lanes, of every length, some without rows or positions."""
    rng = np.random.default_rng(window)
    lens = rng.integers(0, 90, 197).tolist()
    rows = [int(r) if n else 0 for r, n in zip(rng.integers(0, 3, 197), lens)]
    lens[70], rows[70] = 700, 1
    c = Call(4, 2, 64, rows, lens, 16, torch.bfloat16, True, window)
    want = c.run()
    c.check(want)
    c.check(c.run(max_rows=64))
    assert torch.equal(c.run(max_len=100000), want)
    c.cache.status()


@pytest.mark.parametrize("rows,lens", [([1, 1], [130, 77]), ([200, 60], [300, 400])])
def test_guesses_padding_strides(kh, rows, lens):
    """Wrong guesses, rows of no sequence, queries inside a wider row, unaligned ones: the same bits where the cut is the
    same, and the same values everywhere."""
    c = Call(8, 2, 128, rows, lens)
    want = c.run()
    c.check(want)
    for kw in (dict(max_rows=1, max_len=1), dict(max_rows=100000, max_len=2 ** 40), dict(max_rows=0, max_len=0)):
        c.check(c.run(**kw))
    n = sum(rows)
    for shift in (0, 1, 3):
        wide = torch.full(((n + 5) * 12 * 128 + shift,), float("nan"), dtype=torch.bfloat16, device="cuda")[shift:].view(n + 5, 12, 128)
        lse = torch.full((n + 5, 8), float("nan"), device="cuda")
        wide[:n, 2:10], lse[:n] = c.q.cuda(), torch.from_numpy(c.lse).cuda()
        assert torch.equal(c.run(q=wide[:, 2:10], lse=lse), want)
    across = c.q.transpose(0, 1).contiguous().transpose(0, 1).cuda()
    assert torch.equal(c.run(q=across), want)


def test_default_sums_and_log_sum_exps_of_attention(kh):
    """acc of zeros by default; with attention's own log-sum-exps every row's weights add up to one."""
    c = Call(8, 4, 64, [3, 1, 20], [50, 200, 21])
    _, lse = c.cache.attention(c.q.cuda(), c.off, c.len, c.table, return_lse=True)
    acc = c.cache.attention_weights(c.q.cuda(), lse, c.off, c.len, c.table)
    assert acc.shape == (3, 4, c.table.shape[1] * 16)
    # two heads a kv head; lse and the weights are off by some 1e-6 each
    np.testing.assert_allclose(acc.sum(-1).cpu().numpy(), 2.0 * np.array(c.rows)[:, None].repeat(4, 1), rtol=1e-5)
    heads = torch.tensor([[0, 5]] * 24, dtype=torch.int32).cuda()
    _, lse = c.cache.attention(c.q.cuda(), c.off, c.len, c.table, heads=heads, return_lse=True)
    acc = c.cache.attention_weights(c.q.cuda(), lse, c.off, c.len, c.table)
    np.testing.assert_allclose(acc.sum(-1).cpu().numpy(), np.array([[n, 0, n, 0] for n in c.rows]), rtol=1e-5)


@pytest.mark.parametrize("rows", [[1, 1], [100, 70]])
def test_places_that_are_not_there_are_reported(kh, rows):
    from klearu_amd import KlearuError
    c = Call(4, 2, 64, rows, [200, 180])
    want = c.run().cpu()
    c.cache.status()
    t = c.table.clone()
    c.table[1, 3], c.table[1, 7] = c.pages.pages, -5
    got = c.run().cpu()
    with pytest.raises(KlearuError):
        c.cache.status()
    gone = torch.zeros(got.shape[2], dtype=torch.bool)
    gone[48:64] = gone[112:128] = True
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][:, ~gone], want[1][:, ~gone])
    assert torch.equal(got[1][:, gone], c.acc[1][:, gone])
    c.table = t
    short = c.cache.attention_weights(c.q.cuda(), torch.from_numpy(c.lse).cuda(), c.off, c.len, c.table, c.acc[..., :150].contiguous().cuda(),
                                      max_rows=max(rows), max_len=200).cpu()
    with pytest.raises(KlearuError):
        c.cache.status()
    assert torch.equal(short, want[..., :150])
    # pages that no row sees need not be named
    w = Call(4, 2, 64, [1, 1], [200, 180], window=20)
    w.table[0, :11], w.table[1, :10] = -1, 10 ** 6
    w.check(w.run())
    w.cache.status()


def test_other_stream_and_graph(kh):
    c = Call(8, 2, 128, [1, 1, 1], [300, 77, 512])
    want = c.run()
    q, lse, acc = c.q.cuda(), torch.from_numpy(c.lse).cuda(), c.acc.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = c.cache.attention_weights(q, lse, c.off, c.len, c.table, acc.clone(), max_rows=1, max_len=512, stream=s)
    s.synchronize()
    assert torch.equal(got, want)
    p = Call(8, 2, 128, [260, 190], [512, 190])
    for c in (c, p):
        q, lse, start = c.q.cuda(), torch.from_numpy(c.lse).cuda(), c.acc.cuda()
        acc, most = start.clone(), dict(max_rows=max(c.rows), max_len=max(c.lens))
        run = lambda: c.cache.attention_weights(q, lse, c.off, c.len, c.table, acc, **most)  # noqa: E731
        run()
        once = acc.clone()
        run()
        twice = acc.clone()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            run()
        for _ in range(3):
            acc.copy_(start)
            g.replay()
            assert torch.equal(acc, once)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(acc, twice)
            run()

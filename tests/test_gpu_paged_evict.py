"""GPU: eviction from the paged cache and page tables of beams, against plain loops on the host.  Everything is compared
bit for bit: positions are whole numbers, rows move as the codes they are."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, keys, offsets, values

pytestmark = pytest.mark.gpu


def kept_of(w, length, keep, recent, first):
    """The positions that one kv head keeps, ascending."""
    if length <= keep:
        return list(range(length))
    always = set(range(first)) | set(range(length - recent, length))
    rest = [j for j in range(length) if j not in always]
    big = np.where(np.isnan(w), np.inf, w).astype(np.float64)
    rest.sort(key=lambda j: (not np.isnan(w[j]), -big[j], j))
    return sorted(always | set(rest[:keep - len(always)]))


class Cache:
    def __init__(self, kv, dim, lens, page=16, seed=0, spare=1, held=None):
        """Sequences of `held` positions (default: their lengths) in pages of their own."""
        from klearu_amd import paged
        rng = np.random.default_rng(seed + dim)
        held = lens if held is None else held
        self.kv, self.dim, self.lens, self.page, self.held = kv, dim, lens, page, held
        self.pages = Pages(held, page, spare=spare, seed=seed)
        self.c = paged.PagedKv(kv, dim, self.pages.pages, page_size=page)
        n = sum(held)
        self.k, self.v = keys(rng, n, kv, dim), keys(rng, n, kv, dim)
        self.table = self.pages.table.cuda()
        self.len = torch.tensor(lens).cuda()
        self.zero = torch.zeros(len(held), dtype=torch.int64).cuda()
        self.c.append(torch.from_numpy(self.k).cuda(), torch.from_numpy(self.v).cuda(), offsets(held).cuda(), self.zero, self.table)

    def read(self, held=None, table=None):
        held = self.held if held is None else held
        k, v = self.c.gather(offsets(held).cuda(), torch.zeros(len(held), dtype=torch.int64).cuda(), self.table if table is None else table,
                             sum(held))
        cut = np.cumsum([0] + list(held))
        return [(k[a:b].cpu().numpy(), v[a:b].cpu().numpy()) for a, b in zip(cut[:-1], cut[1:])]


def check_evicted(c, before, acc, got, keep, recent, first, lens=None):
    lens = c.lens if lens is None else lens
    kept, left, out = (x.cpu().numpy() for x in got)
    assert kept.dtype == np.int32 and left.tolist() == [min(n, keep) for n in lens]
    after = c.read()
    for b, n in enumerate(lens):
        for h in range(c.kv):
            want = kept_of(acc[b, h], n, keep, recent, first)
            m = len(want)
            assert kept[b, h].tolist() == want + [-1] * (keep - m), (b, h)
            np.testing.assert_array_equal(out[b, h], np.concatenate([acc[b, h][want], np.zeros(acc.shape[2] - m, np.float32)]))
            for x, y in zip(before[b], after[b]):
                np.testing.assert_array_equal(y[:m, h], x[want, h])
                np.testing.assert_array_equal(y[m:, h], x[m:, h])  # what lies behind keeps what it held


def weights(rng, batch, kv, cols, kind):
    w = np.exp(1.5 * rng.standard_normal((batch, kv, cols))).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 4, w.shape).astype(np.float32)
    if kind == "equal":
        w[:] = 0.25
    if kind == "wild":
        w = (rng.standard_normal(w.shape) * 10.0 ** rng.integers(-40, 38, w.shape)).astype(np.float32)
        w[rng.random(w.shape) < 0.05] = np.inf
        w[rng.random(w.shape) < 0.05] = -np.inf
        w[rng.random(w.shape) < 0.1] = 0.0
        w[rng.random(w.shape) < 0.1] = -0.0
        w[rng.random(w.shape) < 0.05] = np.nan
        w[rng.random(w.shape) < 0.02] = -np.float32(np.nan)
    return w


@pytest.mark.parametrize("kv,dim,page", [(1, 64, 16), (3, 128, 32), (2, 256, 64), (4, 64, 256), (8, 128, 16)])
@pytest.mark.parametrize("lens,keep,recent,first", [([100], 64, 10, 4), ([33, 32, 31, 1, 0, 300], 32, 0, 0), ([777, 130], 129, 129, 0),
                                                    ([200, 64], 37, 0, 37), ([500, 90], 1, 0, 0), ([500, 90], 1, 1, 0), ([90], 89, 40, 49)])
@pytest.mark.parametrize("kind", ["plain", "ties"])
def test_evict(kh, kv, dim, page, lens, keep, recent, first, kind):
    rng = np.random.default_rng(keep)
    c = Cache(kv, dim, lens, page)
    acc = weights(rng, len(lens), kv, c.table.shape[1] * page, kind)
    before = c.read()
    for (k, v), a, b in zip(before, np.cumsum([0] + lens), np.cumsum(lens)):
        np.testing.assert_array_equal(k, values(c.k[a:b]).astype(np.float32))
    given = torch.from_numpy(acc).cuda()
    got = c.c.evict(given, c.len, c.table, keep, recent=recent, first=first)
    check_evicted(c, before, acc, got, keep, recent, first)
    np.testing.assert_array_equal(given.cpu().numpy(), acc)
    assert c.len.tolist() == lens
    c.c.status()


@pytest.mark.parametrize("kind", ["wild", "equal", "ties"])
@pytest.mark.parametrize("lens,keep,recent,first", [([4500, 2000], 1500, 100, 3), ([5000], 4999, 0, 0), ([9000, 70], 33, 0, 0)])
@pytest.mark.parametrize("place", [False, True])
def test_orders(kh, kind, lens, keep, recent, first, place):
    """Infinities, NaN, zeros of both signs, many equal weights; into a new tensor and in place."""
    rng = np.random.default_rng(len(kind) + keep)
    c = Cache(2, 64, lens, 64)
    acc = weights(rng, len(lens), 2, c.table.shape[1] * 64, kind)
    before = c.read()
    given = torch.from_numpy(acc).cuda()
    got = c.c.evict(given, c.len, c.table, keep, recent=recent, first=first, out=given if place else None)
    assert (got[2] is given) == place
    check_evicted(c, before, acc, got, keep, recent, first)


@pytest.mark.parametrize("kv,dim,page,length,keep", [(2, 128, 64, 40000, 9000), (1, 64, 16, 70001, 20000), (1, 256, 128, 20000, 19999),
                                                     (1, 64, 32, 16385, 600), (2, 128, 16, 20000, 30000), (1, 64, 16, 9000, 5000)])
@pytest.mark.parametrize("kind", ["plain", "equal", "ties", "wild"])
def test_long(kh, kv, dim, page, length, keep, kind):
    rng = np.random.default_rng(length)
    c = Cache(kv, dim, [length, 1000], page)
    acc = weights(rng, 2, kv, c.table.shape[1] * page, kind)
    before = c.read()
    given = torch.from_numpy(acc).cuda()
    got = c.c.evict(given, c.len, c.table, keep, recent=500, first=4, out=given)
    check_evicted(c, before, acc, got, keep, 500, 4)
    c.c.status()


@pytest.mark.parametrize("lens,keep", [([40000, 0, 9000], 9000), ([20000, 30], 30000), ([16385], 16384)])
@pytest.mark.parametrize("kind", ["plain", "ties"])
def test_long_into_a_new_tensor(kh, lens, keep, kind):
    """The weights go to their places at once where no part still reads what lies there."""
    rng = np.random.default_rng(keep)
    c = Cache(2, 64, lens, 64)
    acc = weights(rng, len(lens), 2, c.table.shape[1] * 64, kind)
    before = c.read()
    given = torch.from_numpy(acc).cuda()
    out = torch.full_like(given, float("nan"))
    got = c.c.evict(given, c.len, c.table, keep, recent=500, first=4, out=out)
    assert got[2] is out and torch.equal(given.cpu(), torch.from_numpy(acc))
    check_evicted(c, before, acc, got, keep, 500, 4)
    c.c.status()


def test_weights_of_other_widths(kh):
    """Wider than the table, as wide as the length, and narrower than it: the positions past them are evicted and reported."""
    from klearu_amd import KlearuError
    rng = np.random.default_rng(1)
    for cols, fine in ((300, True), (200, True), (190, False)):
        c = Cache(2, 128, [200, 20], 16)
        acc = weights(rng, 2, 2, cols, "plain")
        before = c.read()
        got = c.c.evict(torch.from_numpy(acc).cuda(), c.len, c.table, 50, recent=5)
        check_evicted(c, before, acc, got, 50, 5, 0, lens=[min(200, cols), 20])
        if fine:
            c.c.status()
        else:
            with pytest.raises(KlearuError, match="outside its sequence"):
                c.c.status()
    # a table that is shorter than a length; nothing to keep; a negative length
    c = Cache(2, 128, [100, 20], 16)
    acc = weights(rng, 2, 2, 200, "plain")
    before = c.read()
    c.len.copy_(torch.tensor([10 ** 12, -7]))
    got = c.c.evict(torch.from_numpy(acc).cuda(), c.len, c.table, 50, recent=5)
    assert got[1].tolist() == [50, 0] and (got[0][1] == -1).all() and (got[2][1] == 0).all()
    cap = c.table.shape[1] * 16
    assert got[0][0, 0].tolist() == kept_of(acc[0, 0], cap, 50, 5, 0)
    with pytest.raises(KlearuError):
        c.c.status()
    # keeping more than there can be
    c = Cache(2, 128, [100, 20], 16)
    acc = weights(rng, 2, 2, 128, "plain")
    before = c.read()
    check_evicted(c, before, acc, c.c.evict(torch.from_numpy(acc).cuda(), c.len, c.table, 1000, recent=900), 1000, 900, 0)


def test_bad_pages(kh):
    """Positions of pages outside the pool do not move, and nothing is written to them; the others do."""
    from klearu_amd import KlearuError
    rng = np.random.default_rng(9)
    c = Cache(2, 64, [160, 160], 16)
    acc = weights(rng, 2, 2, 176, "plain")
    before = c.read()
    bad = c.table.clone()
    bad[0, 1], bad[0, 4] = c.pages.pages, -1
    kept, left, out = c.c.evict(torch.from_numpy(acc).cuda(), c.len, bad, 60, recent=10)
    with pytest.raises(KlearuError, match="page id"):
        c.c.status()
    after = c.read()
    for b in range(2):
        for h in range(2):
            want = kept_of(acc[b, h], 160, 60, 10, 0)
            assert kept[b, h].tolist() == want
            for x, y in zip(before[b], after[b]):
                w = x[:, h].copy()
                for i, j in enumerate(want):
                    if b == 1 or (j // 16 not in (1, 4) and i // 16 != 1):
                        w[i] = x[j, h]
                np.testing.assert_array_equal(y[:, h], w)


def test_evict_again_and_again(kh):
    """Appended rows and evictions by turns: what is left is what a list on the host would keep."""
    rng = np.random.default_rng(4)
    kv, dim, keep, step = 2, 64, 40, 13
    c = Cache(kv, dim, [53, 30], 16, held=[90, 90])
    cap = c.table.shape[1] * 16
    rows = c.read()
    rows = [[[r[:n, h] for r in rows[b]] for h in range(kv)] for b, n in enumerate(c.lens)]
    acc = torch.zeros(2, kv, cap).cuda()
    lens = torch.tensor(c.lens).cuda()
    for it in range(5):
        n = lens.tolist()
        acc += torch.from_numpy(rng.random((2, kv, cap)).astype(np.float32)).cuda() * (torch.arange(cap).cuda() < lens[:, None, None])
        host = acc.cpu().numpy()
        kept, lens, acc = c.c.evict(acc, lens, c.table, keep, recent=8, first=2, out=acc)
        for b in range(2):
            for h in range(kv):
                want = kept_of(host[b, h], n[b], keep, 8, 2)
                assert kept[b, h].tolist()[:len(want)] == want
                rows[b][h] = [r[want] for r in rows[b][h]]
        k, v = keys(rng, 2 * step, kv, dim), keys(rng, 2 * step, kv, dim)
        c.c.append(torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), offsets([step, step]).cuda(), lens, c.table)
        lens = lens + step
        held = lens.tolist()
        got = c.read(held)
        for b in range(2):
            for h in range(kv):
                for i, x in enumerate((k, v)):
                    rows[b][h][i] = np.concatenate([rows[b][h][i], values(x[b * step:(b + 1) * step, h]).astype(np.float32)])
                    np.testing.assert_array_equal(got[b][i][:, h], rows[b][h][i])
    c.c.status()


# ---------------------------------------------------------------- beams
def tables_of(table, lens, parent, page):
    """The new table and, for each row, the row whose rows it goes on from."""
    batch, beams = parent.shape
    out, source = table.copy(), []
    for b in range(batch):
        free, used = [i for i in range(beams) if i not in parent[b]], set()
        for i, p in enumerate(parent[b]):
            giver = free.pop(0) if p in used else p
            used.add(p)
            w = lens[b] // page
            r = b * beams + i
            out[r, :w], out[r, w:] = table[b * beams + p, :w], table[b * beams + giver, w:]
            source.append(b * beams + p)
    return out, source


@pytest.mark.parametrize("kv,dim,page", [(1, 64, 16), (3, 128, 32), (2, 256, 64), (20, 64, 16), (2, 128, 256)])
@pytest.mark.parametrize("beams,lens", [(1, [37]), (2, [31, 32, 33, 0]), (4, [130, 1, 2, 3, 66]), (7, [200, 15]), (64, [50])])
@pytest.mark.parametrize("kind", ["random", "zero", "turn", "same"])
def test_reorder(kh, kv, dim, page, beams, lens, kind):
    rng = np.random.default_rng(beams)
    batch = len(lens)
    c = Cache(kv, dim, lens, page, spare=2, held=[n + page for n in lens for _ in range(beams)])
    parent = {"random": rng.integers(0, beams, (batch, beams)), "zero": np.zeros((batch, beams), int),
              "turn": np.array([rng.permutation(beams) for _ in lens]), "same": np.arange(beams)[None].repeat(batch, 0)}[kind]
    old, before = c.table.cpu().numpy(), c.read()
    new = c.c.reorder(c.table, c.len, torch.from_numpy(parent.astype(np.int32)).cuda())
    want, source = tables_of(old, lens, parent, page)
    np.testing.assert_array_equal(new.cpu().numpy(), want)
    np.testing.assert_array_equal(c.table.cpu().numpy(), old)
    after = c.read(table=new)
    for r in range(batch * beams):
        n = lens[r // beams]
        for x, y in zip(before[source[r]], after[r]):
            np.testing.assert_array_equal(y[:n], x[:n])
    # what lies behind the sequences' ends in every row's own pages is as it was
    own = {int(p): (r, i) for r in range(batch * beams) for i, p in enumerate(old[r]) if p >= 0}
    for r in range(batch * beams):
        n, w = lens[r // beams], lens[r // beams] // page
        o, i = own[int(want[r, w])]
        for x, y in zip(before[o], after[r]):
            np.testing.assert_array_equal(y[n:(w + 1) * page], x[n:(w + 1) * page])
    c.c.status()


def test_reorder_strides_and_faults(kh):
    from klearu_amd import KlearuError
    c = Cache(2, 64, [40, 50], 16, held=[64] * 6)
    parent = torch.tensor([[2, 2, 0], [1, 1, 1]], dtype=torch.int32).cuda()
    want, _ = tables_of(c.table.cpu().numpy(), [40, 50], parent.cpu().numpy(), 16)
    wide = torch.full((6, c.table.shape[1] + 3), 77, dtype=torch.int32).cuda()
    wide[:, :c.table.shape[1]] = c.table
    out = torch.full_like(wide, 5)
    cols = c.table.shape[1]
    assert c.c.reorder(wide[:, :cols], c.len, parent, out=out[:, :cols]).data_ptr() == out.data_ptr()
    assert (out[:, cols:] == 5).all()
    np.testing.assert_array_equal(out[:, :cols].cpu().numpy(), want)
    c.c.status()
    # a parent that is none: the beam itself
    bad = torch.tensor([[2, 3, 0], [-1, 2, 10 ** 9]], dtype=torch.int32).cuda()
    want, _ = tables_of(c.table.cpu().numpy(), [40, 50], np.array([[2, 1, 0], [0, 2, 2]]), 16)
    np.testing.assert_array_equal(c.c.reorder(c.table, c.len, bad).cpu().numpy(), want)
    with pytest.raises(KlearuError, match="parent"):
        c.c.status()
    # pages outside the pool are listed on, not read or written
    t = c.table.clone()
    t[:, 2] = 10 ** 6
    want, _ = tables_of(t.cpu().numpy(), [40, 50], parent.cpu().numpy(), 16)
    before = c.read()
    np.testing.assert_array_equal(c.c.reorder(t, c.len, parent).cpu().numpy(), want)
    with pytest.raises(KlearuError, match="page id"):
        c.c.status()
    for x, y in zip(before, c.read()):
        np.testing.assert_array_equal(x[0][:32], y[0][:32])
    c.len.copy_(torch.tensor([10 ** 10, -4]))
    c.c.reorder(c.table, c.len, parent)
    with pytest.raises(KlearuError, match="outside its sequence"):
        c.c.status()


def test_streams_and_graphs(kh):
    """On another stream, and captured: replays evict and reorder what lies in the same buffers then."""
    rng = np.random.default_rng(2)
    lens, keep = [300, 90], 64
    c = Cache(2, 64, lens, 16)
    acc = torch.from_numpy(weights(rng, 2, 2, c.table.shape[1] * 16, "plain")).cuda()
    before, raw = c.read(), (torch.from_numpy(c.k).cuda(), torch.from_numpy(c.v).cuda())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = c.c.evict(acc, c.len, c.table, keep, recent=9, stream=s)
    s.synchronize()
    check_evicted(c, before, acc.cpu().numpy(), got, keep, 9, 0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = c.c.evict(acc, c.len, c.table, keep, recent=9)
    for it in range(3):
        acc.copy_(torch.from_numpy(weights(rng, 2, 2, acc.shape[2], "plain")))
        c.c.append(*raw, offsets(lens).cuda(), c.zero, c.table)
        g.replay()
        torch.cuda.synchronize()
        check_evicted(c, before, acc.cpu().numpy(), held, keep, 9, 0)
    r = Cache(2, 64, [45], 16, held=[48] * 4)
    parent = torch.zeros(1, 4, dtype=torch.int32).cuda()
    r.c.reorder(r.table, r.len, parent)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        new = r.c.reorder(r.table, r.len, parent)
    for it in range(3):
        parent.copy_(torch.from_numpy(rng.integers(0, 4, (1, 4))))
        g.replay()
        torch.cuda.synchronize()
        want, _ = tables_of(r.table.cpu().numpy(), [45], parent.cpu().numpy(), 16)
        np.testing.assert_array_equal(new.cpu().numpy(), want)


def test_python_refusals(kh):
    c = Cache(2, 64, [40, 50], 16)
    acc = torch.zeros(2, 2, 80).cuda()
    for bad in (acc[..., ::2], acc.double(), acc[:1], acc[0], acc.cpu()):
        with pytest.raises((ValueError, TypeError)):
            c.c.evict(bad, c.len, c.table, 20)
    with pytest.raises(ValueError, match="out"):
        c.c.evict(acc, c.len, c.table, 20, out=acc[..., :40].contiguous())
    with pytest.raises(ValueError, match="parent"):
        c.c.reorder(c.table, c.len, torch.zeros(2, dtype=torch.int32).cuda())
    with pytest.raises(ValueError, match="table"):
        c.c.reorder(c.table, c.len, torch.zeros(2, 2, dtype=torch.int32).cuda())
    with pytest.raises(ValueError, match="out"):
        c.c.reorder(c.table, c.len, torch.zeros(2, 1, dtype=torch.int32).cuda(), out=c.table[:, :2])

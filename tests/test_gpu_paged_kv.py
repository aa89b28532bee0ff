"""GPU: the paged 4-bit cache, appended rows read back.

The format is a function of the (f32) values, so what is read back is compared bit for bit: against the
definition on the host, and, with a rotation on the way, against appending rows that kh_rope_apply rotated in f32
before."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, keys, offsets, values

pytestmark = pytest.mark.gpu


def cache_of(kv, dim, pages, page):
    from klearu_amd import paged
    return paged.PagedKv(kv, dim, pages, page_size=page)


def same(got, want):
    np.testing.assert_array_equal(got.float().cpu().numpy(), np.asarray(want, np.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv,dim,page", [(1, 64, 16), (3, 128, 32), (2, 256, 64), (5, 64, 256), (1, 128, 16)])
@pytest.mark.parametrize("rows,start", [([1], [0]), ([1, 1, 1], [15, 16, 300]), ([37, 1, 64, 130], [0, 5, 33, 31])])
def test_rows_read_back(kh, dtype, kv, dim, page, rows, start):
    rng = np.random.default_rng(kv * dim + page)
    pg = Pages([r + s for r, s in zip(rows, start)], page)
    c = cache_of(kv, dim, pg.pages, page)
    n = sum(rows)
    k, v = (torch.from_numpy(keys(rng, n, kv, dim)).to(dtype) for _ in range(2))
    off, st, tb = offsets(rows).cuda(), torch.tensor(start).cuda(), pg.table.cuda()
    c.append(k.cuda(), v.cuda(), off, st, tb)
    gk, gv = c.gather(off, st, tb, n)
    same(gk, values(k.float().numpy()))
    same(gv, values(v.float().numpy()))
    bk, bv = c.gather(off, st, tb, n, dtype=torch.bfloat16)
    assert torch.equal(bk, gk.to(torch.bfloat16)) and torch.equal(bv, gv.to(torch.bfloat16))
    # everything before the new rows was never written
    zk, zv = c.gather(offsets(start).cuda(), torch.zeros(len(rows), dtype=torch.int64).cuda(), tb, sum(start))
    # (pages before a sequence's start exist in the table: Pages covers start + rows)
    assert (zk == 0).all() and (zv == 0).all()
    c.status()


def test_neighbours_stay(kh):
    """A position written again changes alone; its neighbours in the page keep their bits."""
    rng = np.random.default_rng(3)
    c = cache_of(2, 128, 4, 16)
    tb = torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda()
    n = 45
    k, v = (torch.from_numpy(keys(rng, n, 2, 128)).cuda() for _ in range(2))
    all_off, zero = offsets([n]).cuda(), torch.zeros(1, dtype=torch.int64).cuda()
    c.append(k, v, all_off, zero, tb)
    for at in (0, 1, 15, 16, 18, 31, 44):
        a, b = (torch.from_numpy(keys(rng, 1, 2, 128) * 3).cuda() for _ in range(2))
        k[at], v[at] = a[0], b[0]
        c.append(a, b, offsets([1]).cuda(), torch.tensor([at]).cuda(), tb)
        gk, gv = c.gather(all_off, zero, tb, n)
        same(gk, values(k.cpu().numpy()))
        same(gv, values(v.cpu().numpy()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (128, 64), (256, 32), (64, 6), (128, 20), (256, 256)])
@pytest.mark.parametrize("own_pos", [False, True])
def test_rotation_on_the_way(kh, dtype, layout, dim, rot, own_pos):
    from klearu_amd import paged
    rng = np.random.default_rng(rot)
    rows, start = [3, 1, 20], [0, 77, 9]
    pg = Pages([r + s for r, s in zip(rows, start)], 16)
    n, kv = sum(rows), 3
    r = paged.Rope(rot, 4000, layout=layout, magnitude=1.1)
    k, v = (torch.from_numpy(keys(rng, n, kv, dim)).to(dtype).cuda() for _ in range(2))
    place = torch.cat([torch.arange(s, s + m) for m, s in zip(rows, start)])
    pos = torch.from_numpy(rng.integers(0, 4000, n)) if own_pos else place
    off, st, tb = offsets(rows).cuda(), torch.tensor(start).cuda(), pg.table.cuda()
    a, b = cache_of(kv, dim, pg.pages, 16), cache_of(kv, dim, pg.pages, 16)
    a.append(k, v, off, st, tb, rope=r, pos=pos.cuda() if own_pos else None)
    b.append(r.apply(k.float(), pos.cuda()), v.float(), off, st, tb)
    for x, y in zip(a.gather(off, st, tb, n), b.gather(off, st, tb, n)):
        assert torch.equal(x, y)


def test_hard_values(kh):
    """All equal, zeros of both signs, subnormals, a huge range, values that are not finite: each group by itself."""
    rng = np.random.default_rng(5)
    x = rng.normal(0, 1, (12, 1, 64)).astype(np.float32)
    x[0, 0, :32] = 0.0
    x[1, 0, :32] = -0.0
    x[2, 0, :32] = 1.0 / 3.0
    x[3, 0, :32] = np.float32(1e-40) * rng.integers(1, 50, 32)
    x[4, 0, 0], x[4, 0, 1] = 3e38, -3e38
    x[5, 0, 7] = np.nan
    x[6, 0, 33] = np.inf
    x[7, 0, 0] = -np.inf
    x[8, 0, :32] = 1000.0 + rng.random(32)
    x[9, 0, :32] = -1000.0 - rng.random(32)
    x[10, 0, 0] = 1e30
    x[11, 0, :32] = np.float32(2.0 ** -126) * rng.random(32)
    x[0, 0, 40] = -np.float32(2.0 ** 100)
    x[1, 0, 40] = np.nextafter(np.float32(2.0 ** 100), np.float32(0))
    c = cache_of(1, 64, 1, 16)
    t, o, z = torch.zeros(1, 1, dtype=torch.int32).cuda(), offsets([12]).cuda(), torch.zeros(1, dtype=torch.int64).cuda()
    xd = torch.from_numpy(x).cuda()
    c.append(xd, xd, o, z, t)
    want = values(x)
    assert np.isnan(want[[4, 5, 7], 0, :32]).all() and np.isnan(want[6, 0, 32:]).all() and np.isfinite(want[6, 0, :32]).all()
    assert np.isnan(want[0, 0, 32:]).all() and np.isfinite(want[1]).all()
    for got in c.gather(o, z, t, 12):
        same(got, want)
        g = got.cpu().numpy()
        fine = np.isfinite(x) & np.isfinite(g)
        from paged_ref import quantize
        s = quantize(x)[1]
        # off by half a step, and by the roundings of a difference, a quotient and a sum
        assert (np.abs(g - x.astype(np.float64))[fine] <= (s / 2 * (1 + 2.0 ** -20) + 2.0 ** -23 * np.abs(x))[fine]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides(kh, dtype, shift):
    """Keys and values inside one projection's rows, heads-first memory and unaligned starts: the same bits."""
    rng = np.random.default_rng(shift)
    n, kv, d = 21, 2, 128
    from klearu_amd import paged
    r = paged.Rope(128, 64)
    buf = torch.zeros(n * 7 * d + shift, dtype=dtype, device="cuda")[shift:].view(n, 7, d)
    buf.copy_(torch.from_numpy(keys(rng, n, 7, d)))
    k, v = buf[:, 3:5], buf[:, 5:]
    o, z, t = offsets([n]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), torch.tensor([[1, 0]], dtype=torch.int32).cuda()
    got = []
    for a, b in ((k, v), (k.contiguous(), v.contiguous()),
                 (k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1))):
        c = cache_of(kv, d, 2, 16)
        c.append(a, b, o, z, t, rope=r)
        got.append(c.gather(o, z, t, n))
    for g in got[1:]:
        assert torch.equal(g[0], got[0][0]) and torch.equal(g[1], got[0][1])


def test_padding_empty_and_bad_places(kh):
    """Rows behind the last sequence and before the first, empty sequences; places and pages that are not there
    are left alone and reported once."""
    from klearu_amd import KlearuError
    rng = np.random.default_rng(9)
    c = cache_of(1, 64, 3, 16)
    k, v = (torch.from_numpy(keys(rng, 10, 1, 64)).cuda() for _ in range(2))
    off = torch.tensor([2, 2, 5, 5, 7]).cuda()  # rows 0, 1 and 7..9 are padding, sequences 0 and 2 empty
    st = torch.tensor([0, 14, 0, 0]).cuda()
    tb = torch.tensor([[-1, -1], [2, 0], [-1, -1], [1, -1]], dtype=torch.int32).cuda()
    c.append(k, v, off, st, tb)
    gk, gv = (torch.full((10, 1, 64), 3.0, device="cuda") for _ in range(2))
    c.gather(off, st, tb, 10, k=gk, v=gv)
    c.status()
    for got, x in ((gk, k), (gv, v)):
        same(got[2:7], values(x[2:7].cpu().numpy()))
        assert (got[:2] == 3).all() and (got[7:] == 3).all()
    before = c.gather(torch.tensor([0, 48]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(),
                      torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), 48)
    for table, start, why in (([[5]], 0, "page id"), ([[-2]], 3, "page id"), ([[1]], 16, "page table"),
                              ([[1]], -1, "page table"), ([[1]], 2 ** 40, "page table")):
        c.append(k[:1], v[:1], offsets([1]).cuda(), torch.tensor([start]).cuda(),
                 torch.tensor(table, dtype=torch.int32).cuda())
        with pytest.raises(KlearuError, match=why):
            c.status()
        c.status()
    after = c.gather(torch.tensor([0, 48]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(),
                     torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), 48)
    assert torch.equal(before[0], after[0]) and torch.equal(before[1], after[1])


def test_rows_without_a_rotation_are_not_appended(kh):
    from klearu_amd import KlearuError, paged
    rng = np.random.default_rng(2)
    c, r = cache_of(1, 64, 1, 16), paged.Rope(64, 8)
    k, v = (torch.from_numpy(keys(rng, 3, 1, 64)).cuda() for _ in range(2))
    o, z, t = offsets([3]).cuda(), torch.zeros(1, dtype=torch.int64).cuda(), torch.zeros(1, 1, dtype=torch.int32).cuda()
    c.append(k, v, o, z, t, rope=r, pos=torch.tensor([7, 8, -1]).cuda())
    gk, gv = c.gather(o, z, t, 3)
    assert (gk[1:] == 0).all() and (gv[1:] == 0).all() and (gv[0] != 0).any()
    c.status()
    with pytest.raises(KlearuError, match="max_pos"):
        r.status()


def test_many_sequences(kh):
    """More sequences than the search stages at once, most of them empty."""
    rng = np.random.default_rng(4)
    rows = (rng.random(3000) < 0.3).astype(int) * rng.integers(1, 4, 3000)
    pg = Pages(list(rows), 16)
    n = int(rows.sum())
    c = cache_of(1, 64, pg.pages, 16)
    k, v = (torch.from_numpy(keys(rng, n, 1, 64)).cuda() for _ in range(2))
    off, st, tb = offsets(rows).cuda(), torch.zeros(3000, dtype=torch.int64).cuda(), pg.table.cuda()
    c.append(k, v, off, st, tb)
    gk, gv = c.gather(off, st, tb, n)
    c.status()
    same(gk, values(k.cpu().numpy()))
    same(gv, values(v.cpu().numpy()))


def test_pool_past_4_gib(kh):
    """Pages on both sides of 2^32 bytes, the last one among them."""
    page, kv, dim = 256, 8, 256
    block = page * dim + page * (dim // 32) * 8
    pages = (1 << 32) // (block * kv) + 40
    rng = np.random.default_rng(8)
    c = cache_of(kv, dim, pages, page)
    tb = torch.tensor([[0, pages - 1, pages - 39, 1]], dtype=torch.int32).cuda()
    n = 4 * page
    k, v = (torch.from_numpy(keys(rng, n, kv, dim)).to(torch.bfloat16).cuda() for _ in range(2))
    o, z = offsets([n]).cuda(), torch.zeros(1, dtype=torch.int64).cuda()
    c.append(k, v, o, z, tb)
    gk, gv = c.gather(o, z, tb, n)
    same(gk, values(k.float().cpu().numpy()))
    same(gv, values(v.float().cpu().numpy()))


@pytest.mark.parametrize("batch", [2, 70])
def test_offsets_past_the_rows(kh, batch):
    """Offsets before the first and past the last row, and past 32 bits: the rows between them, and no others."""
    rng = np.random.default_rng(11)
    c = cache_of(2, 64, 2 * batch, 16)
    k, v = (torch.from_numpy(keys(rng, 9, 2, 64)).cuda() for _ in range(2))
    far = [(-2 ** 40, 5, 2 ** 31), (-2 ** 32 - 5, 9, 2 ** 40), (4, 9, 2 ** 32 + 3), (2 ** 31, 2 ** 31 + 7, 2 ** 33)]
    tb = torch.arange(2 * batch, dtype=torch.int32).view(batch, 2).cuda()
    st = torch.zeros(batch, dtype=torch.int64).cuda()
    for a, b, e in far:
        off = torch.tensor([a, b, e] + [e] * (batch - 2)).cuda()
        c.append(k, v, off, st, tb)
        gk, gv = (torch.full((9, 2, 64), 3.0, device="cuda") for _ in range(2))
        c.gather(off, st, tb, 9, k=gk, v=gv)
        c.status()
        one, two = slice(max(a, 0), min(max(b, 0), 9)), slice(min(b, 9), 9)
        for got, x in ((gk, k), (gv, v)):
            for s in (one, two):
                same(got[s], values(x[s].cpu().numpy()))
            assert (got[: min(max(a, 0), 9)] == 3).all()
        got = c.attention(k.repeat(1, 2, 1), off, torch.full((batch,), 9).cuda(), tb, max_rows=9, max_len=9)
        assert torch.isfinite(got[min(max(a, 0), 9):]).all()
        c.status()

"""GPU: appends and gathers of more rows than one pass of the grid takes, bit for bit against the format."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, keys, offsets, values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kv,dim", [(5, 64), (8, 64), (5, 128), (3, 256)])
@pytest.mark.parametrize("many", [False, True])
def test_rows_past_one_grid(kh, dtype, kv, dim, many):
    """Some 24000 rows: waves take several quads one after the other, and several heads of each (the last unit of an odd
    number of heads is smaller).  A few long sequences, or hundreds (more than 64), some without rows; padding around."""
    from klearu_amd import paged
    rng = np.random.default_rng(kv * dim)
    rows = [int(x) for x in rng.integers(0, 61, 800)] if many else [9001, 0, 14003, 997]
    start = [int(x) for x in rng.integers(0, 9, len(rows))] if many else [3, 0, 30, 17]
    if many:
        rows[5::50] = [0] * len(rows[5::50])
    assert sum(rows) > 23000
    pg = Pages([r + s for r, s in zip(rows, start)], 32)
    n = sum(rows)
    # rows of few distinct patterns: the host's part stays small, and a wave's heads and quads all differ
    base = [torch.from_numpy(keys(rng, 251, kv, dim)).to(dtype) for _ in range(2)]
    at = torch.arange(n) % 251
    c = paged.PagedKv(kv, dim, pg.pages, page_size=32)
    k, v = (torch.full((n + 9, kv, dim), 5.0, dtype=dtype, device="cuda") for _ in range(2))
    k[4:n + 4], v[4:n + 4] = base[0].cuda()[at.cuda()], base[1].cuda()[at.cuda()]
    off, st, tb = offsets(rows).cuda() + 4, torch.tensor(start).cuda(), pg.table.cuda()
    c.append(k, v, off, st, tb)
    gk, gv = (torch.full((n + 9, kv, dim), 3.0, device="cuda") for _ in range(2))
    c.gather(off, st, tb, n + 9, k=gk, v=gv)
    c.status()
    for got, b in ((gk, base[0]), (gv, base[1])):
        want = torch.from_numpy(values(b.float().numpy())).float().cuda()[at.cuda()]
        assert torch.equal(got[4:n + 4], want)
        assert (got[:4] == 3).all() and (got[n + 4:] == 3).all()
    hk, hv = c.gather(off, st, tb, n + 9, dtype=torch.bfloat16)
    assert torch.equal(hk[4:n + 4], gk[4:n + 4].to(torch.bfloat16)) and torch.equal(hv[4:n + 4], gv[4:n + 4].to(torch.bfloat16))


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("kv,dim,rot", [(5, 64, 64), (5, 128, 64), (3, 256, 20)])
def test_rotated_rows_past_one_grid(kh, layout, kv, dim, rot):
    """The same with a rotation on the way: the bits of rows that were rotated before."""
    from klearu_amd import paged
    rows, start = [12007, 13002], [1, 40]
    n = sum(rows)
    pg = Pages([r + s for r, s in zip(rows, start)], 64)
    r = paged.Rope(rot, 20000, layout=layout)
    torch.manual_seed(rot)
    k, v = (torch.randn(n, kv, dim, device="cuda") for _ in range(2))
    pos = torch.cat([torch.arange(s, s + m) for m, s in zip(rows, start)]).cuda()
    off, st, tb = offsets(rows).cuda(), torch.tensor(start).cuda(), pg.table.cuda()
    a, b = (paged.PagedKv(kv, dim, pg.pages, page_size=64) for _ in range(2))
    a.append(k, v, off, st, tb, rope=r)
    b.append(r.apply(k, pos), v, off, st, tb)
    for x, y in zip(a.gather(off, st, tb, n), b.gather(off, st, tb, n)):
        assert torch.equal(x, y)
    a.status()
    r.status()

"""GPU: rotations by positions along several axes, against 64 bits (tolerances as for one axis: three roundings of
2^-24 for each product, BF16 outputs rounded by 2^-8 once more), against the rotation of one axis, and taken back."""
import numpy as np
import pytest
import torch

from paged_ref import Pages, keys, offsets
from test_gpu_rope import bound, check

pytestmark = pytest.mark.gpu


def frequencies(sections, restart, theta=10000.0):
    half = sum(sections)
    if not restart:
        return theta ** (-np.arange(half) / half)
    return np.concatenate([theta ** (-np.arange(n) / n) for n in sections])


def rotated(x, pos, sections, restart, layout, transpose=False, mag=1.0):
    """x [rows, heads, dim] f64, pos [axes, rows] -> (y, tolerance without the output's rounding)."""
    axis = np.repeat(np.arange(len(sections)), sections)
    a = pos[axis].T.astype(np.float64) * frequencies(sections, restart)
    c, s = (mag * np.cos(a))[:, None], (mag * np.sin(a))[:, None] * (-1.0 if transpose else 1.0)
    h = len(axis)
    i0, i1 = (np.arange(h), np.arange(h) + h) if layout == 0 else (2 * np.arange(h), 2 * np.arange(h) + 1)
    y, tol = x.copy(), np.zeros_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    tol[..., i0] = tol[..., i1] = 3 * 2.0 ** -24 * mag * (np.abs(x[..., i0]) + np.abs(x[..., i1]))
    return y, tol


SHAPES = [(1, 1, 64, (16, 16)), (7, 3, 128, (16, 24, 24)), (33, 5, 96, (8, 8, 8, 8)), (9, 2, 72, (18, 18)), (5, 4, 128, (1, 40, 7)),
          (4, 3, 33, (2, 1, 3)), (130, 1, 256, (32, 64, 16, 16)), (6, 2, 80, (20,))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,sections", SHAPES)
@pytest.mark.parametrize("restart,transpose", [(False, False), (True, False), (False, True), (True, True)])
def test_rotation(kh, dtype, layout, rows, heads, dim, sections, restart, transpose):
    from klearu_amd import paged
    rng = np.random.default_rng(rows * dim)
    rot, axes = 2 * sum(sections), len(sections)
    x = torch.from_numpy(rng.normal(0, 1, (rows, heads, dim)).astype(np.float32)).to(dtype)
    pos = rng.integers(0, 900, (axes, rows))
    pos[:, -1] = 899
    r = paged.Rope(rot, 900, layout=layout, sections=sections, restart=restart, magnitude=1.25)
    p = torch.from_numpy(pos if axes > 1 else pos[0]).cuda()
    y = r.apply(x.cuda(), p, transpose=transpose)
    want, tol = rotated(x.double().numpy(), pos, sections, restart, layout, transpose, 1.25)
    check(y, want, bound(want, tol, dtype))
    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
    z = x.cuda()
    assert torch.equal(r.apply(z, p, out=z, transpose=transpose), y)  # in place
    # unaligned: another kernel, the same bits
    w = torch.zeros(rows * heads * dim + 1, dtype=dtype, device="cuda")[1:].view(rows, heads, dim)
    w.copy_(x)
    assert torch.equal(r.apply(w, p, transpose=transpose), y)
    r.status()


@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("sections", [(16, 24, 24), (5, 30, 29)])
def test_equal_positions_are_one_axis(kh, layout, sections):
    """Text: the same position along every axis is the rotation of one axis, bit for bit."""
    from klearu_amd import paged
    x = torch.randn(50, 4, 128, device="cuda")
    pos = torch.randint(0, 5000, (50,), device="cuda")
    one, many = paged.Rope(128, 5000, layout=layout), paged.Rope(128, 5000, layout=layout, sections=sections)
    assert torch.equal(one.apply(x, pos), many.apply(x, pos.expand(3, 50).contiguous()))


@pytest.mark.parametrize("sections,layout", [((16, 16), 0), ((3, 20, 9), 1)])
def test_gradient(kh, sections, layout):
    """The transposed rotation is the gradient: against <g, R(x + d) - R(x - d)> / 2 (the rotation is linear, so
    differences of any size give it), summed in 64 bits; both sides are off by 3 * 2^-24 of products of up to 64 elements' sums."""
    from klearu_amd import paged
    r = paged.Rope(64, 100, layout=layout, sections=sections)
    torch.manual_seed(0)
    x, g, d = (torch.randn(20, 2, 64, device="cuda") for _ in range(3))
    pos = torch.randint(0, 100, (len(sections), 20), device="cuda")
    back = r.apply(g, pos, transpose=True)
    left = ((r.apply(x + d, pos).double() - r.apply(x - d, pos).double()) / 2 * g.double()).sum(-1)
    right = (back.double() * d.double()).sum(-1)
    size = 6 * 2.0 ** -24 * ((g.abs().sum(-1) * (x.abs() + d.abs()).max(-1).values * 2) + back.abs().sum(-1) * d.abs().max(-1).values)
    assert ((left - right).abs() <= size).all()
    both = r.apply(r.apply(x, pos), pos, transpose=True)  # R^T R = 1
    np.testing.assert_allclose(both.cpu().numpy(), x.cpu().numpy(), rtol=0, atol=12 * 2.0 ** -24 * 2 * float(x.abs().max()))


@pytest.mark.parametrize("sections", [(16, 16), (7, 25)])
@pytest.mark.parametrize("layout", [0, 1])
def test_padding_and_far_positions(kh, sections, layout):
    """A negative position along any axis: padding.  One past the table: reported, unless the row is padding."""
    from klearu_amd import KlearuError, paged
    r = paged.Rope(64, 50, layout=layout, sections=sections)
    x = torch.randn(6, 2, 64, device="cuda")
    pos = torch.tensor([[0, -1, 3, 49, 60, 5], [1, 2, -2, 49, -1, 6]]).cuda()
    out = torch.full_like(x, 7.0)
    r.apply(x, pos, out=out)
    r.status()
    assert (out[[1, 2, 4]] == 7).all() and (out[[0, 3, 5]] != 7).any()
    want, tol = rotated(x[[0, 3, 5]].double().cpu().numpy(), pos[:, [0, 3, 5]].cpu().numpy(), sections, False, layout)
    check(out[[0, 3, 5]], want, tol)
    pos[1, 5] = 50
    out.fill_(7.0)
    r.apply(x, pos, out=out)
    with pytest.raises(KlearuError, match="position"):
        r.status()
    assert (out[[1, 2, 4, 5]] == 7).all()
    for bad in (pos[0], pos.T.contiguous(), pos.to(torch.int32)):
        with pytest.raises((ValueError, TypeError)):
            r.apply(x, bad)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("dim,sections", [(64, (16, 16)), (128, (16, 24, 24)), (128, (5, 30, 29)), (256, (8, 8, 4, 4)), (64, (3, 4))])
@pytest.mark.parametrize("own_pos", [False, True])
def test_rotation_on_the_way_into_the_cache(kh, dtype, layout, dim, sections, own_pos):
    """append with a rotation of several axes against rows that were rotated before."""
    from klearu_amd import KlearuError, paged
    rng = np.random.default_rng(dim)
    rows, start = [3, 1, 20], [0, 77, 9]
    pg = Pages([r + s for r, s in zip(rows, start)], 16)
    n, kv, axes = sum(rows), 3, len(sections)
    r = paged.Rope(2 * sum(sections), 4000, layout=layout, sections=sections, magnitude=1.1)
    k, v = (torch.from_numpy(keys(rng, n, kv, dim)).to(dtype).cuda() for _ in range(2))
    place = torch.cat([torch.arange(s, s + m) for m, s in zip(rows, start)])
    pos = torch.from_numpy(rng.integers(0, 4000, (axes, n))) if own_pos else place.expand(axes, n).contiguous()
    off, st, tb = offsets(rows).cuda(), torch.tensor(start).cuda(), pg.table.cuda()
    a, b = paged.PagedKv(kv, dim, pg.pages, page_size=16), paged.PagedKv(kv, dim, pg.pages, page_size=16)
    a.append(k, v, off, st, tb, rope=r, pos=pos.cuda() if own_pos else None)
    b.append(r.apply(k.float(), pos.cuda()), v.float(), off, st, tb)
    for x, y in zip(a.gather(off, st, tb, n), b.gather(off, st, tb, n)):
        assert torch.equal(x, y)
    r.status()
    if own_pos:  # a bad position along one axis: the row is not appended at all
        bad = pos.clone()
        bad[axes - 1, 4], bad[0, 9] = 4000, -1
        want = a.gather(off, st, tb, n)
        a.append(k + 1, v + 1, off, st, tb, rope=r, pos=bad.cuda())
        with pytest.raises(KlearuError):
            r.status()
        for x, y in zip(a.gather(off, st, tb, n), want):
            assert torch.equal(x[[4, 9]], y[[4, 9]]) and not torch.equal(x[3], y[3])
    with pytest.raises(ValueError):
        a.append(k, v, off, st, tb, rope=r, pos=pos[0].cuda())

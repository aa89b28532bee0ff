"""GPU: kh_rope_apply against the rotation in 64 bits.

y0 = x0 c - x1 s and y1 = x1 c + x0 s with c, s rounded to f32: three roundings of 2^-24 for each product
(the factor's, its own, the sum's), so y is off by at most 3 * 2^-24 (|x0| + |x1|) magnitude; BF16 outputs are
rounded once more, by 2^-8 of themselves."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def frequencies(rot, theta=10000.0, scaling=0, factor=1.0, original=0, low=1.0, high=32.0):
    f = []
    for i in range(rot // 2):
        base = theta * factor ** (rot / (rot - 2)) if scaling == 2 else theta
        x = base ** (-2.0 * i / rot)
        if scaling == 1:
            x /= factor
        if scaling == 3:
            g = min(1.0, max(0.0, (original * x / (2 * math.pi) - low) / (high - low)))
            x *= g + (1 - g) / factor
        f.append(x)
    return np.array(f)


def rotated(x, pos, f, layout, mag=1.0, transpose=False):
    """x [rows, heads, dim] f64 -> (y, tolerance without the output's rounding)."""
    a = pos.astype(np.float64)[:, None] * f[None]
    c, s = (mag * np.cos(a))[:, None], (mag * np.sin(a))[:, None] * (-1.0 if transpose else 1.0)
    h = len(f)
    i0, i1 = (np.arange(h), np.arange(h) + h) if layout == 0 else (2 * np.arange(h), 2 * np.arange(h) + 1)
    y, tol = x.copy(), np.zeros_like(x)
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i1] * c + x[..., i0] * s
    tol[..., i0] = tol[..., i1] = 3 * 2.0 ** -24 * mag * (np.abs(x[..., i0]) + np.abs(x[..., i1]))
    return y, tol


def check(got, want, tol):
    got = got.double().cpu().numpy()
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), float(off.max())


def bound(want, tol, dtype):
    return tol + (2.0 ** -8 * np.abs(want) * (1 + 2.0 ** -8) + 2.0 ** -8 * tol if dtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 1, 64, 64), (1, 32, 128, 128), (7, 3, 128, 64), (129, 5, 64, 16),
                                                (33, 2, 256, 256), (5, 3, 80, 80), (4, 7, 96, 24), (3, 2, 72, 10),
                                                (6, 1, 2, 2), (2, 3, 33, 6)])
@pytest.mark.parametrize("transpose", [False, True])
def test_rotation(kh, dtype, layout, rows, heads, dim, rot, transpose):
    from klearu_amd import paged
    rng = np.random.default_rng(rows * dim + rot)
    x = torch.from_numpy(rng.normal(0, 1, (rows, heads, dim)).astype(np.float32)).to(dtype)
    pos = rng.integers(0, 5000, rows)
    pos[-1] = 4999
    r = paged.Rope(rot, 5000, layout=layout, magnitude=1.25)
    y = r.apply(x.cuda(), torch.from_numpy(pos).cuda(), transpose=transpose)
    assert y.dtype == dtype and y.shape == x.shape
    want, tol = rotated(x.double().numpy(), pos, frequencies(rot), layout, 1.25, transpose)
    check(y, want, bound(want, tol, dtype))
    assert torch.equal(y[..., rot:].cpu(), x[..., rot:])
    r.status()


@pytest.mark.parametrize("scaling,kw", [(1, dict(factor=8.0)), (2, dict(factor=4.0)),
                                        (3, dict(factor=16.0, original_len=4096)),
                                        (3, dict(factor=8.0, original_len=8192, low=1.0, high=4.0))])
def test_scaled_for_far_positions(kh, scaling, kw):
    from klearu_amd import paged
    rng = np.random.default_rng(scaling)
    n, last = 64, 262143
    x = torch.from_numpy(rng.normal(0, 1, (n, 2, 128)).astype(np.float32))
    pos = np.concatenate([rng.integers(0, last + 1, n - 2), [0, last]])
    r = paged.Rope(128, last + 1, scaling=scaling, theta=500000.0, **kw)
    f = frequencies(128, 500000.0, scaling, kw["factor"], kw.get("original_len", 0), kw.get("low", 1.0),
                    kw.get("high", 32.0))
    want, tol = rotated(x.double().numpy(), pos, f, 0)
    check(r.apply(x.cuda(), torch.from_numpy(pos).cuda()), want, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_strides_and_in_place(kh, dtype, layout, shift):
    """Heads inside a wider projection row, [heads, rows] memory, unaligned starts; into another buffer
    and in place.  Every layout of memory gives the packed call's bits, and nothing else changes."""
    from klearu_amd import paged
    rng = np.random.default_rng(shift)
    n, h, d = 9, 4, 128
    r = paged.Rope(96, 64, layout=layout)
    pos = torch.arange(n, device="cuda") * 3
    x = torch.from_numpy(rng.normal(0, 1, (n, h, d)).astype(np.float32)).to(dtype).cuda()
    want = r.apply(x, pos)
    wide = torch.full((n * (h + 2) * d + shift,), 7.0, dtype=dtype, device="cuda")[shift:].view(n, h + 2, d)
    wide[:, 1:h + 1] = x
    assert torch.equal(r.apply(wide[:, 1:h + 1], pos), want)
    across = torch.zeros((h * n * d + shift,), dtype=dtype, device="cuda")[shift:].view(h, n, d).transpose(0, 1)
    assert r.apply(x, pos, out=across) is across and torch.equal(across, want)
    r.apply(wide[:, 1:h + 1], pos, out=wide[:, 1:h + 1])
    assert torch.equal(wide[:, 1:h + 1], want)
    assert (wide[:, 0] == 7).all() and (wide[:, h + 1:] == 7).all()
    one = x[:1, :1].expand(n, h, d)  # strides of zero, read only
    assert torch.equal(r.apply(one, pos), r.apply(one.contiguous(), pos))


def test_padding_far_rows_and_no_rows(kh):
    from klearu_amd import KlearuError, paged
    r = paged.Rope(64, 10)
    x = torch.randn(4, 2, 64, device="cuda")
    out = torch.full_like(x, 5.0)
    pos = torch.tensor([3, -1, 9, -7], device="cuda")
    r.apply(x, pos, out=out)
    r.status()
    assert (out[1] == 5).all() and (out[3] == 5).all() and torch.equal(out[:1], r.apply(x[:1], pos[:1]))
    r.apply(x, torch.tensor([0, 10, 2 ** 40, 1], device="cuda"), out=out)
    assert (out[1] == 5).all() and torch.equal(out[0], x[0])
    with pytest.raises(KlearuError, match="max_pos"):
        r.status()
    r.status()
    assert r.apply(x[:0], pos[:0]).shape == (0, 2, 64)


@pytest.mark.parametrize("layout", [0, 1])
def test_gradient(kh, layout):
    """The transposed rotation is the gradient: against differences of y = R x (linear: a central
    difference is exact but for the roundings) and against <R x, g> = <x, R^T g>."""
    from klearu_amd import paged
    rng = np.random.default_rng(layout)
    n, h, d = 3, 2, 64
    r = paged.Rope(48, 100, layout=layout, magnitude=1.1)
    pos = torch.tensor([0, 17, 99], device="cuda")
    x, g = (torch.from_numpy(rng.normal(0, 1, (n, h, d)).astype(np.float32)).cuda() for _ in range(2))
    back = r.apply(g, pos, transpose=True).double()
    a, b = (r.apply(x, pos).double() * g.double()).sum(), (x.double() * back).sum()
    size = 1.1 * (x.double().abs() * g.double().abs()).sum() * 2 * 6 * 2.0 ** -24
    assert abs(float(a - b)) <= float(size) * 2
    for _ in range(6):
        t, i, e = int(rng.integers(n)), int(rng.integers(h)), int(rng.integers(d))
        up, down = x.clone(), x.clone()
        up[t, i, e] = 1.0
        down[t, i, e] = -1.0
        diff = ((r.apply(up, pos).double() - r.apply(down, pos).double()) * g.double()).sum() / 2
        near = 8 * 2.0 ** -24 * 1.1 * float((x[t, i].abs().max() + 1) * g[t, i].abs().max()) * 4
        assert abs(float(diff - back[t, i, e])) <= near


def test_stream_and_graph(kh):
    """Captured on a side stream and replayed with other rows and positions between eager calls."""
    from klearu_amd import paged
    r = paged.Rope(128, 4096)
    x = torch.randn(5, 8, 128, device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(5, device="cuda")
    y = torch.empty_like(x)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        r.apply(x, pos, out=y)
    side = torch.cuda.Stream()
    for k in range(4):
        x.copy_(torch.randn(5, 8, 128, device="cuda"))
        pos.copy_(torch.randint(0, 4096, (5,), device="cuda"))
        g.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        z = r.apply(x, pos, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(y, z) and torch.equal(y, r.apply(x, pos))

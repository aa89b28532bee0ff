"""GPU: continuations of beams against 64 bits.

A score is f64 and rounded to f32 once: 2^-24 of itself.  Its log-sum-exp is off by what the f32 exponentials are off,
at most 2^-21 of each.  Within a beam continuations are compared by their logits, so they come exactly; between beams
two whose scores are nearer than those errors may change places."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def scores_of(x, s, done, end):
    """All continuations' scores [batch, beams * vocab], f64, as the definition has them."""
    x = x.astype(np.float64)
    batch, beams, vocab = x.shape
    y = np.full(x.shape, -np.inf)
    for b in range(batch):
        for i in range(beams):
            if not np.isfinite(s[b, i]):
                continue
            if done is not None and done[b, i]:
                y[b, i, end] = s[b, i]
                continue
            top = x[b, i].max()
            with np.errstate(all="ignore"):
                log = np.log(np.exp(x[b, i] - top).sum())
            if np.isfinite(top) and np.isfinite(log):  # beside a `top` of 1e38 the logarithm would be lost, to 64 bits too
                y[b, i] = np.float64(s[b, i]) + ((x[b, i] - top) - log)
    return y.reshape(batch, -1)


def check(got, x, s, k, done=None, end=0):
    y, i, v = (t.cpu().numpy() for t in got)
    batch, beams, vocab = x.shape
    assert y.shape == i.shape == v.shape == (batch, k) and i.dtype == v.dtype == np.int32
    ref = scores_of(x, s, done, end)
    for b in range(batch):
        order = np.lexsort((np.arange(beams * vocab), -ref[b]))[:k]
        flat = i[b].astype(np.int64) * vocab + v[b]
        assert (i[b] >= 0).all() and (i[b] < beams).all() and (v[b] >= 0).all() and (v[b] < vocab).all()
        assert len(set(flat.tolist())) == k
        want = ref[b][order]
        fine = np.isfinite(want)
        np.testing.assert_array_equal(np.isfinite(y[b]), fine)
        assert (y[b][~fine] == -np.inf).all()
        tol = 2.0 ** -21 + 2.0 ** -24 * np.abs(want[fine])
        assert (np.abs(y[b][fine] - want[fine]) <= tol).all(), b
        # the same continuations, but for beams that lie closer than the tolerance
        for r in np.nonzero(flat != order)[0]:
            assert i[b, r] != order[r] // vocab and abs(ref[b][flat[r]] - want[r]) <= 2.0 ** -20, (b, r)


def logits(rng, batch, beams, vocab):
    x = rng.normal(0, 2.5, (batch, beams, vocab)) + 6 * (rng.random((batch, beams, vocab)) < 20 / vocab)
    return x.astype(np.float32), (-20 * rng.random((batch, beams))).astype(np.float32)


def run(x, s, k, done=None, end=0, dtype=torch.float32):
    from klearu_amd import beam
    t = torch.from_numpy(x).to(dtype)
    got = beam.select(t.cuda(), torch.from_numpy(s).cuda(), k, None if done is None else torch.from_numpy(done).cuda(), end)
    return t.float().numpy(), got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,k", [(1, 1, 1, 1), (1, 4, 32000, 8), (3, 1, 17, 17), (2, 8, 8191, 16), (1, 3, 50, 64),
                                                 (5, 2, 4097, 3), (1, 64, 1000, 64), (2, 5, 131, 11), (1, 2, 131071, 5)])
@pytest.mark.parametrize("ends", [False, True])
def test_select(kh, dtype, batch, beams, vocab, k, ends):
    rng = np.random.default_rng(vocab + k)
    x, s = logits(rng, batch, beams, vocab)
    done, end = (rng.random((batch, beams)) < 0.4, vocab // 2) if ends else (None, 0)
    xs, got = run(x, s, k, done, end, dtype)
    check(got, xs, s, k, done, end)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,beams,vocab,k", [(1100, 4, 1500, 5), (260, 4, 5000, 9), (30, 7, 20000, 33)])
def test_many_rows(kh, dtype, batch, beams, vocab, k):
    """Rows that one wave takes, or some of a block, or all."""
    rng = np.random.default_rng(batch)
    x, s = logits(rng, batch, beams, vocab)
    xs, got = run(x, s, k, dtype=dtype)
    check(got, xs, s, k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [6, 40])
def test_runs_are_alike(kh, dtype, k):
    """What waves of a row hear of each other, and when, does not change the result: many equal logits, run after run."""
    from klearu_amd import beam
    rng = np.random.default_rng(k)
    x, s = logits(rng, 20, 4, 60000)
    xd, sd = torch.from_numpy(np.floor(4 * x) / 4).to(dtype).cuda(), torch.from_numpy(s).cuda()
    want = beam.select(xd, sd, k)
    check(want, xd.float().cpu().numpy(), s, k)
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(beam.select(xd, sd, k), want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_first_step_and_all_ended(kh, dtype):
    rng = np.random.default_rng(0)
    x, s = logits(rng, 3, 4, 5000)
    s[:, 1:] = -np.inf
    xs, got = run(x, s, 8, dtype=dtype)
    check(got, xs, s, 8)
    assert (got[1] == 0).all()
    done = np.ones((3, 4), bool)
    for end in (0, 3, 4999):
        xs, got = run(x, s, 8, done, end, dtype)
        check(got, xs, s, 8, done, end)
    xs, got = run(x[:, :1], s[:, :1], 6, done[:, :1], 2, dtype)
    check(got, xs, s[:, :1], 6, done[:, :1], 2)


@pytest.mark.parametrize("vocab", [40, 4096, 20000])
@pytest.mark.parametrize("kind", ["equal", "few", "zeros", "masked"])
def test_ties(kh, vocab, kind):
    """Many equal logits: the first by (beam, token)."""
    rng = np.random.default_rng(vocab)
    x, s = logits(rng, 2, 3, vocab)
    if kind == "equal":
        x[:] = 1.5
        s[:] = -2.0
    if kind == "few":
        x = np.floor(x / 3).astype(np.float32)
    if kind == "zeros":
        x = np.where(rng.random(x.shape) < 0.5, np.float32(0.0), np.float32(-0.0))
    if kind == "masked":
        x[rng.random(x.shape) < 0.9995] = -np.inf
        x[..., 7] = 0
    for k in (1, 7, 64):
        xs, got = run(x, s, k)
        check(got, xs, s, k)
        for b in range(2):  # equal logits of one beam are neighbours, in the order of their tokens
            y, i, v = (t[b].cpu().numpy() for t in got)
            for r in range(1, k):
                if i[r] == i[r - 1] and y[r] > -np.inf and xs[b, i[r], v[r]] == xs[b, i[r - 1], v[r - 1]]:
                    assert v[r] > v[r - 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,left", [(3000, 5), (40000, 3), (40000, 20000), (40000, 0)])
def test_masks(kh, dtype, vocab, left):
    """Masked tokens at -inf or at the type's lowest value; all but a few, all of a beam, the first or the last ones."""
    rng = np.random.default_rng(left)
    for low in (-np.inf, float(torch.finfo(dtype).min)):
        x, s = logits(rng, 2, 3, vocab)
        for b in range(2):
            for i in range(3):
                gone = rng.permutation(vocab)[left:] if i < 2 else np.arange(vocab)[-(vocab - left):]
                x[b, i, gone] = low
        for k in (4, 17, 64):
            xs, got = run(x, s, k, dtype=dtype)
            check(got, xs, s, k)


@pytest.mark.parametrize("vocab", [5000, 70000])
@pytest.mark.parametrize("way", ["up", "down", "steps", "late"])
@pytest.mark.parametrize("k", [1, 16, 31, 64])
def test_orders_of_logits(kh, vocab, way, k):
    """Logits that rise or fall along the vocabulary (every next one is a better one), in steps of equal ones, or far
    larger at the end."""
    rng = np.random.default_rng(k)
    x, s = logits(rng, 1, 2, vocab)
    x = np.sort(x, -1)
    if way == "down":
        x = x[..., ::-1].copy()
    if way == "steps":
        x = np.floor(x * 2).astype(np.float32)
    if way == "late":
        x[..., -vocab // 3:] += 500
        x[..., -3:] += 5e4
    xs, got = run(x, s, k)
    check(got, xs, s, k)


def test_nan_among_others(kh):
    """A beam with NaN here and there has no continuation, however many there are; its neighbours lose nothing."""
    rng = np.random.default_rng(4)
    x, s = logits(rng, 2, 4, 9000)
    x[0, 1][rng.random(9000) < 0.9] = np.nan
    x[0, 2, 1:] = np.nan
    x[1, 3][rng.random(9000) < 0.3] = -np.float32(np.nan)
    x[1, 0, 17] = np.nan
    for k in (8, 64):
        xs, got = run(x, s, k)
        check(got, xs, s, k)
        assert not np.isin(got[1][0].cpu().numpy(), (1, 2)).any() and not np.isin(got[1][1].cpu().numpy(), (0, 3)).any()


def test_values_that_are_not_finite(kh):
    """NaN or +inf among a beam's logits, or nothing but -inf: it has no continuation.  So has one whose score is not finite."""
    rng = np.random.default_rng(3)
    x, s = logits(rng, 1, 8, 9000)
    x[0, 0, 8999], x[0, 1, 0], x[0, 2], x[0, 3, 4000:8200] = np.nan, np.inf, -np.inf, np.nan
    s[0, 4], s[0, 5], s[0, 6] = np.nan, np.inf, -np.inf
    xs, got = run(x, s, 12)
    check(got, xs, s, 12)
    assert (got[1] == 7).all()
    x[0, 7] = np.nan
    xs, got = run(x, s, 12)
    check(got, xs, s, 12)
    assert (got[0] == -np.inf).all() and (got[1] == 0).all() and got[2][0].tolist() == list(range(12))
    x, s = logits(rng, 1, 2, 100)
    x *= 1e30
    xs, got = run(x, s, 5)
    check(got, xs, s, 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shift,gap", [(0, 0), (1, 0), (3, 5), (0, 1), (7, 8)])
def test_strides(kh, dtype, shift, gap):
    """Rows apart, and starting anywhere between two 16-byte borders: the bits of the packed call's."""
    from klearu_amd import beam
    rng = np.random.default_rng(shift + gap)
    batch, beams, vocab, k = 2, 3, 4133, 9
    x, s = logits(rng, batch, beams, vocab)
    packed = torch.from_numpy(x).to(dtype).cuda()
    want = beam.select(packed, torch.from_numpy(s).cuda(), k)
    check(want, packed.float().cpu().numpy(), s, k)
    wide = torch.full((batch * beams * (vocab + gap) + shift,), float("nan"), dtype=dtype, device="cuda")[shift:]
    wide = wide.view(batch, beams, vocab + gap)
    wide[..., :vocab] = packed
    got = beam.select(wide[..., :vocab], torch.from_numpy(s).cuda(), k)
    # chunks begin at 16-byte borders, so that sums differ in their last bits
    check(got, packed.float().cpu().numpy(), s, k)


def test_refusals_stream_and_graph(kh):
    from klearu_amd import KlearuError, beam
    rng = np.random.default_rng(8)
    x, s = logits(rng, 2, 4, 3000)
    xd, sd = torch.from_numpy(x).cuda(), torch.from_numpy(s).cuda()
    for args in ((xd[..., ::2], sd, 4), (xd.transpose(0, 1), sd.T.contiguous(), 4), (xd, sd[:, :3], 4), (xd, sd.double(), 4),
                 (xd.half(), sd, 4), (xd[0], sd, 4), (xd, sd.cpu(), 4)):
        with pytest.raises((ValueError, TypeError)):
            beam.select(*args)
    for k, end in ((0, 0), (65, 0), (4, 3000), (4, -1)):
        with pytest.raises(KlearuError):
            beam.select(xd, sd, k, torch.zeros(2, 4, dtype=torch.bool).cuda(), end)
    want = beam.select(xd, sd, 8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = beam.select(xd, sd, 8, stream=st)
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        held = beam.select(xd, sd, 8)
    for it in range(3):
        x, s = logits(rng, 2, 4, 3000)
        xd.copy_(torch.from_numpy(x))
        sd.copy_(torch.from_numpy(s))
        g.replay()
        torch.cuda.synchronize()
        check(held, x, s, 8)
        assert all(torch.equal(a, b) for a, b in zip(held, beam.select(xd, sd, 8)))

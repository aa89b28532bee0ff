"""GPU: the order of continuations whose scores are equal, or come out equal.

Scores are compared in f64 as they are computed.  Beams of the same logits and score have the same scores, bit for bit, wherever
their rows start, so that the order between them is that of the beams; within a beam larger logits come first, also where
the score has no digits for the difference, and equal ones by their tokens.  Every place is known, without a tolerance."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("beams,vocab,k", [(8, 131071, 16), (8, 20001, 20), (3, 4133, 9), (8, 1025, 8), (5, 1021, 64), (8, 77, 33)])
@pytest.mark.parametrize("seed", range(4))
def test_beams_that_are_alike(kh, dtype, beams, vocab, k, seed):
    """Rows of odd lengths: each starts elsewhere between two 16-byte borders."""
    from klearu_amd import beam
    rng = np.random.default_rng(seed)
    row = rng.normal(0, 2.5, vocab) + 6 * (rng.random(vocab) < 20 / vocab)
    x = torch.from_numpy(np.tile(row.astype(np.float32), (2, beams, 1))).to(dtype)
    s = torch.full((2, beams), -7.25)
    y, i, v = (t.cpu() for t in beam.select(x.cuda(), s.cuda(), k))
    best = np.lexsort((np.arange(vocab), -x[0, 0].double().numpy()))
    # the best logit of every beam, then the next one of every beam; equal logits by beams first
    want = sorted(((-x[0, 0, t].item(), b, t) for t in best[:k] for b in range(beams)))[:k]
    for b in range(2):
        assert i[b].tolist() == [w[1] for w in want]
        assert v[b].tolist() == [w[2] for w in want]
        for logit in {w[0] for w in want}:
            assert len({y[b, r].item() for r, w in enumerate(want) if w[0] == logit}) == 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,shift", [(4133, 0), (4133, 3), (131071, 1), (900, 5)])
def test_bits_do_not_depend_on_where_rows_start(kh, dtype, vocab, shift):
    from klearu_amd import beam
    rng = np.random.default_rng(vocab + shift)
    x = torch.from_numpy(rng.normal(0, 2.5, (2, 3, vocab)).astype(np.float32)).to(dtype).cuda()
    s = torch.from_numpy((-20 * rng.random((2, 3))).astype(np.float32)).cuda()
    wide = torch.empty(2, 3, (vocab + 15) // 8 * 8, dtype=dtype, device="cuda")[..., :vocab]  # all rows at a border
    wide.copy_(x)
    odd = torch.empty(6 * vocab + shift, dtype=dtype, device="cuda")[shift:].view(2, 3, vocab)
    odd.copy_(x)
    want = beam.select(wide, s, 9)
    for got in (beam.select(x, s, 9), beam.select(odd, s, 9)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [200, 5000, 70001])
@pytest.mark.parametrize("top,small", [(1e20, 1.0), (5.0, 2.0 ** -70)])
def test_logits_that_the_scores_do_not_tell_apart(kh, dtype, vocab, top, small):
    """One logit far larger than the steps between the others: they are in their own order all the same."""
    from klearu_amd import beam
    rng = np.random.default_rng(vocab)
    x = np.full((1, 2, vocab), -small * 300, np.float32)
    at = np.stack([rng.permutation(vocab)[:121] for _ in range(2)])
    for b in range(2):
        x[0, b, at[b, :120]] = small * rng.permutation(np.arange(1, 121))
        x[0, b, at[b, 120]] = top
    s = np.array([[-20.0, -21.0 - 2.0 * top]], np.float32)  # the second beam's scores all lie below the first one's
    for k in (3, 16, 64):
        y, i, v = (t[0].cpu().numpy() for t in beam.select(torch.from_numpy(x).to(dtype).cuda(), torch.from_numpy(s).cuda(), k))
        assert (i == 0).all() and v.tolist() == np.argsort(-x[0, 0], kind="stable")[:k].tolist()

"""GPU: a decoder's steps together: beams over a shared paged cache whose keys turn by positions along three axes, attention,
its weights, eviction, selection and reordering, step after step, against lists on the host; and captured in a graph.

Eviction writes to pages, so those must be a beam's own: either the budget is less than a page, or nothing is
evicted and whole pages are shared, or every beam goes on from itself."""
import numpy as np
import pytest
import torch

from paged_ref import keys, offsets, values
from test_gpu_beam import check as check_beams
from test_gpu_paged_evict import kept_of, tables_of

pytestmark = pytest.mark.gpu
BATCH, BEAMS, HEADS, KV, DIM, PAGE, VOCAB = 2, 3, 4, 2, 64, 16, 500
ROWS = BATCH * BEAMS


class Decoder:
    """Rows (beams) with tables of their own pages; rows of one sequence are equally long."""

    def __init__(self, cols=8, seed=0):
        from klearu_amd import paged
        rng = np.random.default_rng(seed)
        self.cache = paged.PagedKv(KV, DIM, ROWS * cols, page_size=PAGE)
        self.rope = paged.Rope(DIM, 1000, sections=(8, 12, 12))
        self.table = torch.from_numpy(rng.permutation(ROWS * cols).astype(np.int32).reshape(ROWS, cols)).cuda()
        self.one = offsets([1] * ROWS).cuda()
        self.q, self.k, self.v = (torch.zeros(ROWS, n, DIM, device="cuda") for n in (HEADS, KV, KV))
        self.pos = torch.zeros(3, ROWS, dtype=torch.int64, device="cuda")
        self.lens = torch.zeros(ROWS, dtype=torch.int64, device="cuda")
        self.acc = torch.zeros(ROWS, KV, cols * PAGE, device="cuda")
        self.logits, self.scores = torch.zeros(BATCH, BEAMS, VOCAB, device="cuda"), torch.zeros(BATCH, BEAMS, device="cuda")

    def step(self, keep, recent, branch=True):
        from klearu_amd import beam
        c = self.cache
        c.append(self.k, self.v, self.one, self.lens, self.table, rope=self.rope, pos=self.pos)
        lens = self.lens + 1
        q = self.rope.apply(self.q, self.pos)
        y, lse = c.attention(q, self.one, lens, self.table, return_lse=True, max_rows=1)
        c.attention_weights(q, lse, self.one, lens, self.table, self.acc, max_rows=1)
        kept, lens, _ = c.evict(self.acc, lens, self.table, keep, recent=recent, out=self.acc)
        s, parent, token = beam.select(self.logits, self.scores, BEAMS)
        if not branch:
            parent.copy_(torch.arange(BEAMS, dtype=torch.int32, device="cuda").expand(BATCH, BEAMS))
        table = c.reorder(self.table, lens[::BEAMS].contiguous(), parent)
        row = (parent.long() + torch.arange(BATCH, device="cuda")[:, None] * BEAMS).flatten()
        self.table.copy_(table)
        self.acc.copy_(self.acc[row])
        self.lens.copy_(lens)
        self.scores.copy_(s)
        return y, kept, s, parent, token

    def set(self, it, rng):
        for t in (self.q, self.k, self.v):
            t.copy_(torch.from_numpy(keys(rng, ROWS, t.shape[1], DIM)))
        self.pos.copy_(torch.tensor([[it], [it // 4], [it % 4]]).expand(3, ROWS))
        self.logits.copy_(torch.from_numpy(rng.normal(0, 2, (BATCH, BEAMS, VOCAB)).astype(np.float32)))


WAYS = [(12, 4, True), (1000, 8, True), (24, 8, False)]


@pytest.mark.parametrize("keep,recent,branch", WAYS)
def test_steps(kh, keep, recent, branch):
    """40 steps: outputs within the tolerances of the pieces, kept positions and cached rows exactly."""
    rng = np.random.default_rng(1)
    d = Decoder()
    held = [[(np.zeros((0, DIM)), np.zeros((0, DIM))) for _ in range(KV)] for _ in range(ROWS)]  # per row and kv head
    sums = [[np.zeros(0) for _ in range(KV)] for _ in range(ROWS)]
    for it in range(40):
        d.set(it, rng)
        q = d.rope.apply(d.q, d.pos).double().cpu().numpy()
        k, v = values(d.rope.apply(d.k, d.pos).cpu().numpy()), values(d.v.cpu().numpy())
        logits, before, scores = d.logits.cpu().numpy(), d.table.cpu().numpy(), d.scores.cpu().numpy()
        y, kept, s, parent, token = d.step(keep, recent, branch)
        acc = d.acc.cpu().numpy()
        y, kept = y.double().cpu().numpy(), kept.cpu().numpy()
        if branch:
            check_beams((s, parent, token), logits, scores, BEAMS)
        par = parent.cpu().numpy()
        for r in range(ROWS):
            for h in range(KV):
                K, V = (np.concatenate([a, b[r, h][None]]) for a, b in zip(held[r][h], (k, v)))
                w = np.concatenate([sums[r][h], [0.0]])
                for g in range(HEADS // KV):
                    x = K @ q[r, h * 2 + g] * DIM ** -0.5
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    w = w + p
                    np.testing.assert_allclose(y[r, h * 2 + g], p @ V, rtol=0, atol=2e-5 * np.abs(V).max())
                n = len(w)
                mine = kept[r, h][kept[r, h] >= 0]
                # by the weights of the host; nearer ones than their errors may change places
                order = kept_of(w.astype(np.float32), n, keep, recent, 0)
                if mine.tolist() != order:
                    odd = sorted(set(order) ^ set(mine.tolist()))
                    assert np.ptp(w[odd]) <= 1e-5 * w[odd].max(), (it, r, h)
                held[r][h], sums[r][h] = (K[mine], V[mine]), w[mine]
        want, source = tables_of(before, [len(sums[b * BEAMS][0]) for b in range(BATCH)], par, PAGE)
        np.testing.assert_array_equal(d.table.cpu().numpy(), want)
        held, sums = [list(held[r]) for r in source], [list(sums[r]) for r in source]
        n = len(sums[0][0])
        assert d.lens.tolist() == [n] * ROWS
        gk, gv = d.cache.gather(offsets([n] * ROWS).cuda(), torch.zeros(ROWS, dtype=torch.int64).cuda(), d.table, n * ROWS)
        for r in range(ROWS):
            for h in range(KV):
                for x, z in zip((gk, gv), held[r][h]):
                    np.testing.assert_array_equal(x[r * n:(r + 1) * n, h].cpu().numpy(), z.astype(np.float32))
                np.testing.assert_allclose(acc[r, h, :n], sums[r][h], rtol=1e-5)
                assert (acc[r, h, n:] == 0).all()
    d.cache.status()
    d.rope.status()


@pytest.mark.parametrize("keep,recent,branch", WAYS)
def test_steps_in_a_graph(kh, keep, recent, branch):
    """The same step captured once and replayed, beside the eager one: the same bits throughout."""
    a, b = Decoder(seed=3), Decoder(seed=3)
    ra, rb = np.random.default_rng(5), np.random.default_rng(5)
    for it in range(3):
        a.set(it, ra)
        b.set(it, rb)
        a.step(keep, recent, branch)
        b.step(keep, recent, branch)
    g = torch.cuda.CUDAGraph()
    a.set(3, ra)
    b.set(3, rb)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        held = a.step(keep, recent, branch)
    for it in range(3, 40):
        if it > 3:
            a.set(it, ra)
            b.set(it, rb)
        g.replay()
        want = b.step(keep, recent, branch)
        for x, y in zip(held, want):
            assert torch.equal(x, y), it
        for x, y in zip((a.table, a.acc, a.lens, a.scores), (b.table, b.acc, b.lens, b.scores)):
            assert torch.equal(x, y), it
    a.cache.status()

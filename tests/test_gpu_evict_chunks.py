"""GPU: kept positions that one block moves in several chunks, each over places that the chunk before has just filled from.

A block of a kv head takes 2048 positions at a time (1024 at 256-wide heads) through its registers, where no more than that
is kept or there are 64 kv heads; the same sizes at fewer heads go through the workspace.  Everything is compared
bit for bit."""
import numpy as np
import pytest
import torch

from test_gpu_paged_evict import Cache, check_evicted, weights

pytestmark = pytest.mark.gpu


def rising(rng, batch, kv, cols):
    """The last positions are the heaviest: everything moves by all that is evicted."""
    return np.tile(np.arange(cols, dtype=np.float32), (batch, kv, 1)) + rng.random((batch, kv, 1)).astype(np.float32)


def sparse(rng, batch, kv, cols):
    """Light positions are rare, so that most positions move by a few places."""
    w = 1 + rng.random((batch, kv, cols)).astype(np.float32)
    w[rng.random(w.shape) < 0.002] = 0
    return w


@pytest.mark.parametrize("place", [False, True])
@pytest.mark.parametrize("kind", ["plain", "rising", "sparse"])
@pytest.mark.parametrize("kv,dim,page,lens,keep,recent,first", [
    (2, 256, 64, [4000], 1025, 0, 0), (2, 256, 16, [4001, 3100], 3001, 100, 3), (1, 256, 128, [3010], 3002, 7, 0),
    (1, 128, 64, [4500, 2050], 2049, 0, 0), (3, 128, 16, [5000], 4095, 500, 4), (2, 128, 32, [4110], 4094, 0, 16),
    (3, 64, 16, [4400, 2052, 100], 2050, 1, 1), (1, 64, 256, [4300], 4093, 0, 0), (2, 64, 64, [4099], 4096, 4000, 0),
    (1, 64, 64, [17000], 4095, 33, 5), (1, 256, 64, [16500], 2047, 0, 0), (3, 256, 32, [2047, 2000], 1999, 4, 700)])
def test_several_chunks(kh, kv, dim, page, lens, keep, recent, first, kind, place):
    rng = np.random.default_rng(keep + dim)
    c = Cache(kv, dim, lens, page)
    size = (len(lens), kv, c.table.shape[1] * page)
    acc = rising(rng, *size) if kind == "rising" else sparse(rng, *size) if kind == "sparse" else weights(rng, *size, "plain")
    before = c.read()
    given = torch.from_numpy(acc).cuda()
    got = c.c.evict(given, c.len, c.table, keep, recent=recent, first=first, out=given if place else None)
    check_evicted(c, before, acc, got, keep, recent, first)
    c.c.status()


@pytest.mark.parametrize("kind", ["plain", "rising", "sparse"])
@pytest.mark.parametrize("kv,dim,page,lens,keep", [(16, 64, 16, [2600, 2051, 2500, 2100, 2600, 2055, 2300, 2599], 2050),
                                                   (128, 64, 64, [4500], 4203), (64, 128, 32, [2200, 2100], 2051), (128, 256, 16, [1100], 1026),
                                                   (64, 64, 256, [4300], 4093), (64, 128, 16, [2400], 2050), (32, 256, 64, [2500, 2100], 2049)])
def test_many_heads(kh, kv, dim, page, lens, keep, kind):
    rng = np.random.default_rng(keep + kv)
    c = Cache(kv, dim, lens, page)
    size = (len(lens), kv, c.table.shape[1] * page)
    acc = rising(rng, *size) if kind == "rising" else sparse(rng, *size) if kind == "sparse" else weights(rng, *size, "plain")
    before = c.read()
    got = c.c.evict(torch.from_numpy(acc).cuda(), c.len, c.table, keep, recent=200, first=2)
    check_evicted(c, before, acc, got, keep, 200, 2)
    c.c.status()


def test_again_and_again(kh):
    """A cache that is cut, grows by the next positions and is cut again, as a decoder's does."""
    rng = np.random.default_rng(5)
    c = Cache(2, 128, [4600], 64, held=[4600])
    acc = torch.zeros(1, 2, c.table.shape[1] * 64, device="cuda")
    lens, keep = c.len, 4094
    for n in (4600, 4096, 4107, 4095):
        lens = torch.tensor([n]).cuda()
        w = weights(rng, 1, 2, acc.shape[2], "plain")
        before = c.read()
        acc.copy_(torch.from_numpy(w))
        got = c.c.evict(acc, lens, c.table, keep, recent=64, out=acc)
        check_evicted(c, before, w, got, keep, 64, 0, lens=[n])
    c.c.status()

"""GPU: attention weights where a wave or a block goes on past what it looked up first: pages of more steps than a wave has
lanes, and more blocks of rows than it has lanes.  References and tolerances are those of the other sizes."""
import pytest
import torch

from test_gpu_paged_weights import Call

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 16), (2, 1, 128, 32), (2, 2, 256, 64)])
@pytest.mark.parametrize("rows,lens,window", [([1], [5200], 0), ([1, 1, 1], [700, 9001, 4100], 0), ([1, 1], [5200, 9001], 4999)])
def test_few_rows_many_steps(kh, dtype, heads, kv, dim, page, rows, lens, window):
    """A guess of one position leaves four waves: some forty steps and more each, where a wave looks 32 up at once."""
    c = Call(heads, kv, dim, rows, lens, page, dtype, True, window)
    c.check(c.run(max_len=1))
    c.check(c.run())
    c.cache.status()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads,kv,dim,page,length", [(8, 1, 64, 16, 9000), (8, 1, 128, 32, 10000), (8, 2, 256, 64, 5000)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 8999)])
def test_many_rows_many_steps(kh, dtype, heads, kv, dim, page, length, causal, window):
    """The guess makes it one share, which takes more than 64 steps."""
    c = Call(heads, kv, dim, [20], [length], page, dtype, causal, window)
    c.check(c.run(max_len=1))
    c.check(c.run())
    c.cache.status()


@pytest.mark.parametrize("heads,kv,dim,dtype,rows,lens,window", [
    (16, 1, 256, torch.float32, [600], [600], 0), (16, 1, 256, torch.float32, [600, 530], [900, 530], 0),
    (16, 1, 256, torch.float32, [700], [700], 33), (16, 1, 64, torch.bfloat16, [2100], [2100], 0)])
def test_many_blocks_of_rows(kh, heads, kv, dim, dtype, rows, lens, window):
    """More than 64 blocks of rows (of 128 rows times heads, 512 in the last case): shares begin among the later ones."""
    c = Call(heads, kv, dim, rows, lens, 64, dtype, True, window)
    c.check(c.run())
    c.check(c.run(max_len=1))
    c.cache.status()

"""GPU: rotations past the 2^32 threads of one launch, against small calls of the same rows and against 64 bits."""
import numpy as np
import pytest
import torch

from test_gpu_rope import check, frequencies, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory():
    """40 GiB of device memory, which other tests' cached blocks do not hold, and this one's do not stay."""
    torch.cuda.empty_cache()
    if torch.cuda.is_available() and torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GiB of device memory")
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("layout", [0, 1])
def test_rows_past_one_launch(kh, layout):
    """A pair a thread (two elements a head are no 16-byte piece): 2^32 + 3 * 2^12 pairs, 16 GiB of BF16."""
    from klearu_amd import paged
    rows, heads, period = 2 ** 20 + 3, 2 ** 12, 7
    r = paged.Rope(2, period, layout=layout)
    few = torch.randn(period, heads, 2, device="cuda").to(torch.bfloat16)
    want = r.apply(few, torch.arange(period, device="cuda"))
    x = torch.empty(rows, heads, 2, dtype=torch.bfloat16, device="cuda")
    cut = rows - rows % period
    x[:cut].view(-1, period, heads, 2).copy_(few)
    x[cut:] = few[: rows - cut]
    pos = torch.arange(rows, device="cuda") % period
    assert r.apply(x, pos, out=x) is x
    assert bool((x[:cut].view(-1, period, heads, 2) == want).all()) and torch.equal(x[cut:], want[: rows - cut])
    r.status()


def test_table_past_one_launch(kh):
    """2^32 + 64 pairs of cosines and sines, 32 GiB: positions at both ends of the table and around 2^32 pairs."""
    from klearu_amd import paged
    most = 2 ** 26 + 1
    r = paged.Rope(128, most)
    pos = np.array([0, 1, 12345, 2 ** 25 + 3, most - 3, most - 2, most - 1])
    x = torch.from_numpy(np.random.default_rng(1).normal(0, 1, (len(pos), 2, 128)).astype(np.float32))
    want, tol = rotated(x.double().numpy(), pos, frequencies(128), 0)
    # an angle of 2^26 turns by 2^-27 of a radian where its f64 product and frequency are off by 2^-53 each
    tol = tol + 2.0 ** -26 * np.abs(x.double().numpy()).max()
    check(r.apply(x.cuda(), torch.from_numpy(pos).cuda()), want, tol)

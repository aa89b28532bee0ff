"""GPU: what status() reports, call after call and from a stream that does not wait for the null stream."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_records_right_after_a_report(kh):
    """A report clears the record before a call behind it, on another stream, can set it again."""
    from klearu_amd import KlearuError, paged
    c, r = paged.PagedKv(1, 64, 1, page_size=16), paged.Rope(64, 8)
    x = torch.zeros(1, 1, 64, device="cuda")
    off, start = torch.tensor([0, 1], device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
    bad, far = torch.tensor([[7]], dtype=torch.int32, device="cuda"), torch.tensor([8], device="cuda")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(200):
        c.append(x, x, off, start, bad, stream=side)
        with pytest.raises(KlearuError, match="page id"):
            c.status()
        r.apply(x, far, stream=side)
        with pytest.raises(KlearuError, match="max_pos"):
            r.status()
    c.status()
    r.status()

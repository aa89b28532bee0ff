"""CPU: results that lie partly on what a call still reads are refused, before any device call."""
import pytest
import torch  # noqa: F401 (skipif)

from klearu_amd import _lib
from test_paged_args import ARG, P, cache, change, refused

BIG = 1 << 30  # addresses that are never followed


def passes(name, args):
    """The call gets as far as the device: nothing in its arguments is refused (there is no GPU at these addresses)."""
    lib = _lib.load()
    assert getattr(lib, name)(*args) != ARG, lib.kh_last_error()


EVICT = dict(c=cache(), acc=BIG, acols=100, len=P, batch=3, table=P, cols=8, ts=8, keep=40, recent=10, first=4, kept=P,
             out=BIG, left=2 * P, ws=P, wsb=1 << 40, st=None)
ACC = 3 * 2 * 100 * 4  # bytes of the weights


@pytest.mark.parametrize("acols", [100, 100000])  # in one block, in parts
def test_eviction_into_a_part_of_its_weights(acols):
    size = ACC * acols // 100
    for by in (4, -4, 2 * acols * 4, -2 * acols * 4, size - 4, 4 - size):
        refused("kh_paged_kv_evict", change(EVICT, acols=acols, out=BIG + by), ARG, "overlap")
    for by in (3, -8, 16, 20, -20):  # three lengths of eight bytes each
        refused("kh_paged_kv_evict", change(EVICT, acols=acols, left=P + by), ARG, "place of their own")


@pytest.mark.skipif("torch.cuda.is_available()", reason="the calls that pass would run")
def test_evictions_that_pass():
    for by in (0, ACC, -ACC):
        passes("kh_paged_kv_evict", change(EVICT, out=BIG + by))
    for by in (24, -24):
        passes("kh_paged_kv_evict", change(EVICT, left=P + by))

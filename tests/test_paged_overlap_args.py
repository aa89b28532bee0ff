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


REORDER = dict(c=cache(), table=BIG, cols=8, ts=20, len=P, batch=2, beams=4, parent=P, out=2 * BIG, os=20, st=None)


def test_reordering_onto_its_table():
    """Rows of eight columns, twenty apart."""
    for by in (0, 4 * 7, -4 * 7, 4 * 13, -4 * 13, 4 * 20, -4 * 20, 4 * 140, 4 * 147, -4 * 147, 4 * 132 + 4):
        refused("kh_paged_kv_reorder", change(REORDER, out=BIG + by), ARG, "place of its own")
    # other distances: row 2 of one lies in row 1 of the other
    refused("kh_paged_kv_reorder", change(REORDER, os=10, out=BIG), ARG, "place of its own")
    refused("kh_paged_kv_reorder", change(REORDER, os=10, out=BIG + 8 * 4), ARG, "place of its own")
    refused("kh_paged_kv_reorder", change(REORDER, ts=8, os=8, out=BIG + 63 * 4), ARG, "place of its own")


@pytest.mark.skipif("torch.cuda.is_available()", reason="the calls that pass would run")
def test_reorderings_that_pass():
    """The two tables in the rows of one buffer, after each other, or in turn."""
    for by in (4 * 8, 4 * 12, -4 * 8, -4 * 12, 4 * 148, -4 * 148, 4 * 160, 4 * 8 + 2 * 4 * 20):
        passes("kh_paged_kv_reorder", change(REORDER, out=BIG + by))
    passes("kh_paged_kv_reorder", change(REORDER, ts=40, os=20, cols=8, batch=1, beams=2, out=BIG + 4 * 10))
    passes("kh_paged_kv_reorder", change(REORDER, ts=8, os=8, out=BIG + 64 * 4))


def test_rows_past_any_address():
    for kw in (dict(ts=2 ** 62), dict(os=2 ** 62), dict(ts=2 ** 58, os=2 ** 58)):
        refused("kh_paged_kv_reorder", change(REORDER, **kw), ARG, "apart")

"""CPU: which way evicted sequences go, as the workspace that is asked for tells: images of pages where positions are copied out
and back, none where a block moves a kv head's positions by itself."""
import ctypes as C

import pytest

from klearu_amd import _lib
from test_paged_args import CacheHandle, P


@pytest.mark.parametrize("batch,kv,keep,copies", [(1, 8, 2048, False), (1, 8, 2049, True), (2, 31, 4096, True), (1, 32, 2049, True),
                                                  (2, 32, 2049, False), (1, 64, 9000, False), (63, 1, 2100, True), (1, 8, 10000, False)])
def test_few_heads_that_keep_much_are_copied(batch, kv, keep, copies):
    lib, need = _lib.load(), C.c_int64(-1)
    cache = CacheHandle(kv, 64, 16, 4, 10, 1280, 0, P, P)
    assert lib.kh_paged_kv_evict_workspace(C.byref(cache), batch, keep, 10000, C.byref(need)) == 0
    assert need.value == (batch * kv * -(-keep // 16) * 1280 if copies else 0)

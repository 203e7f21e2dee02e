"""The page pool under a request that grows for long, host side (no GPU)."""
import ctypes as C
import time

import zinc_amd
from zinc_amd import KvPagePool


def test_a_request_that_grows_by_a_page_at_a_time():
    """400000 pages: 0.4 s; 10 to 45 s where each call copies the request's list."""
    n = 400000
    pool, page = KvPagePool(n, 16), C.c_uint32()
    alloc, ref = zinc_amd.lib().zh_kv_pool_alloc, C.byref(page)
    t = time.perf_counter()
    for i in range(n):
        assert alloc(pool.h, 1, 1, ref) == 0 and page.value == n - 1 - i
    assert time.perf_counter() - t < 4
    assert pool.free_count() == 0 and pool.pages(1).tolist() == list(range(n - 1, -1, -1))

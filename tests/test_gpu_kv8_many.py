"""Attention over the 8-bit cache for batches of many sequences, one of them long: each
dealt out in the two ways."""
import numpy as np
import pytest
from test_gpu_kv8 import E4M3, Cache, attend, close, ctx, expect, tables_for, tolerance, zh  # noqa: F401
from test_gpu_kv8_edges import starts_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("n,long,nkv,hd,G,rows", [(800, 30000, 8, 64, 1, 1), (1700, 9000, 8, 64, 2, 1), (800, 27000, 2, 128, 4, 1),
                                                  (300, 9000, 4, 64, 2, 9), (4000, 2000, 1, 64, 1, 1)])
def test_one_long_among_many_short(zh, ctx, n, long, nkv, hd, G, rows, t):  # noqa: F811
    rng = np.random.default_rng(n)
    lens = rows + rng.integers(0, 60, n)
    lens[n // 3] = long
    tables, total = tables_for(rng, lens, 2)
    cache = Cache(ctx, rng, total, nkv, hd, E4M3)
    counts = [rows] * n
    starts = None if rows == 1 else starts_of(counts)
    q, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts)
    s = np.unique(np.concatenate([[0, n // 3 - 1, n // 3, n // 3 + 1, n - 1], rng.integers(0, n, 60)]))
    row = (s[:, None] * rows + np.arange(rows)).ravel()
    want, *terms = expect(cache, tables[s], q[row], [rows] * len(s), lens[s], hd ** -0.5)
    close(got[row], want, tolerance(cache, t, want, *terms, lens, floor=-39))

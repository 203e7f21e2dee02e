"""Pages of the 8-bit cache that are continued step by step: the codes are exactly those of
the plain form iterated in the same order, whichever form of the write takes a row and
whatever else is in its call; how far values are off then, and written in one call."""
import kv8_ref as ref
import numpy as np
import pytest
from test_gpu_kv8 import E4M3, I8, Cache, ctx, u32, zh  # noqa: F401
from test_gpu_kv8_edges import caches_agree, starts_of, stored, write

pytestmark = pytest.mark.gpu


def rows_of(rng, kind, n, heads, hd):
    """Rows that grow by the token (a page's scale rises often), and shrink, jump or stay."""
    x = rng.normal(size=(n, heads, hd))
    t = np.arange(n)[:, None, None]
    size = {"growing": 1.25 ** (t % 16 + t // 16), "doubling": 2.0 ** (t % 16), "jumping": 2.0 ** rng.integers(-9, 10, (n, heads, 1)),
            "shrinking": 0.8 ** t, "level": np.ones_like(t)}[kind]
    return (x * size).astype(np.float32)


def values(cache, got, tables, length):
    """k and v [2][kv heads][length][hd], and their blocks' scales [2][kv heads][length][1]."""
    p = np.arange(length)
    at, pages = tables[0, p // 16].astype(np.int64) * 16 + p % 16, tables[0, p // 16]
    s = np.stack([got[2 + i][pages].T[..., None].astype(np.float64) for i in (0, 1)])
    return np.stack([ref.decode(got[i][:, at], cache.fmt) for i in (0, 1)]) * s, s


@pytest.mark.parametrize("steps", [[1] * 45, [3, 1, 7, 1, 1, 16, 2, 5, 9], [45]], ids=["rows", "chunks", "once"])
@pytest.mark.parametrize("kind", ["growing", "doubling", "jumping", "shrinking", "level"])
@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_pages_written_in_steps(zh, ctx, fmt, kind, steps):  # noqa: F811
    """Rounded once, a value is off by half a step; continued, by less than one step of the
    last scale (i8), or half a step of its own and less than 2^-9 of the scale (e4m3)."""
    rng = np.random.default_rng(len(kind) + len(steps))
    nq, nkv, hd, n = 2, 2, 64, sum(steps)
    x = rows_of(rng, kind, n, nq + 2 * nkv, hd)
    tables = u32([[2, 0, 1]])
    cache = Cache(ctx, rng, 3, nkv, hd, fmt)
    done = 0
    for c in steps:
        done += c
        kv = cache.batch(zh, tables, [done], None if c == 1 else [0, c])
        write(zh, ctx, kv, x[done - c:done], nq, nkv, hd, check=False)
        cache.k, cache.v, cache.ks, cache.vs = stored(cache, tables, [c], [done], x[done - c:done], nq)
    ctx.sync()
    got = cache.get()
    caches_agree(cache, got, (cache.k, cache.v, cache.ks, cache.vs))
    y, s = values(cache, got, tables, n)
    v = np.stack([x[:, nq:nq + nkv], x[:, nq + nkv:]]).astype(np.float64).transpose(0, 2, 1, 3)
    err = np.abs(y - v)
    if len(steps) == 1:
        assert (err <= (0.5 * s if fmt == I8 else np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10 * s))).all()
    else:
        assert (err < s).all() if fmt == I8 else (err <= np.abs(v) * 2.0 ** -4 + 2.0 ** -9 * s).all()


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("nq,nkv,hd,rd", [(4, 2, 128, 128), (5, 5, 64, 32), (8, 1, 128, 24)])
def test_both_forms_of_the_write_leave_the_same_bytes(zh, ctx, fmt, t, nq, nkv, hd, rd):  # noqa: F811
    """The same single rows, step by step: as a row a sequence, as rows of pages, and beside
    other sequences' chunks; codes and scales bit for bit, q the same to its rounding."""
    rng = np.random.default_rng(nq * hd + t)
    S, steps = 5, 20
    past = np.array([0, 3, 15, 30, 31])
    dtype = (np.float32, np.float16)[t]
    size = np.dtype(dtype).itemsize
    tables = u32(rng.permutation(3 * 4 * S).reshape(3 * S, 4))  # (the last 2 S sequences': the others of the third way)
    caches = [Cache(ctx, np.random.default_rng(9), 3 * 4 * S, nkv, hd, fmt) for _ in range(3)]
    freq, w = (1e6 ** (-np.arange(0, rd, 2) / rd)).astype(np.float32), (1 + 0.2 * rng.normal(size=hd)).astype(np.float32)
    more = dict(inv_freq=ctx.upload(freq), rope_dim=rd, q_norm_w=ctx.upload(w), k_norm_w=ctx.upload(w), eps=1e-6)
    width = nq + 2 * nkv
    for i in range(steps):
        x = (rng.normal(size=(S, width, hd)) * 1.4 ** (i % 16)).astype(dtype)
        lens = past + i + 1
        q0 = ctx.alloc(S * nq * hd * size)
        write(zh, ctx, caches[0].batch(zh, tables[:S], lens), x, nq, nkv, hd, check=False, q_out=q0, **more)
        q1 = ctx.alloc(S * nq * hd * size)
        write(zh, ctx, caches[1].batch(zh, tables[:S], lens, starts_of([1] * S)), x, nq, nkv, hd, check=False, q_out=q1, **more)
        # others of many rows before and after
        counts = [7] * S + [1] * S + [11] * S
        y = rng.normal(size=(sum(counts), width, hd)).astype(dtype)
        y[7 * S:8 * S] = x
        q2 = ctx.alloc(len(y) * nq * hd * size)
        order = np.concatenate([np.arange(S, 2 * S), np.arange(S), np.arange(2 * S, 3 * S)])
        write(zh, ctx, caches[2].batch(zh, tables[order], np.concatenate([lens + 7, lens, lens + 11]), starts_of(counts)), y,
              nq, nkv, hd, check=False, q_out=q2, **more)
        a, b, c = (q.download(dtype, S * nq * hd, off) for q, off in ((q0, 0), (q1, 0), (q2, 7 * S * nq * hd * size)))
        assert np.array_equal(b, c)
        # (a sum of squares in another order, a rounding of the angle's sine: 2^-19 of a pair, and the store's)
        tol = 2.0 ** -19 * np.abs(b.astype(np.float64)).reshape(S * nq, hd).max(1, keepdims=True) * 2
        d = np.abs(a.astype(np.float64) - b.astype(np.float64)).reshape(S * nq, hd)
        assert (d <= tol + np.abs(b.astype(np.float64)).reshape(S * nq, hd) * (0 if t == 0 else 2.0 ** -10)).all()
    ctx.sync()
    pages = np.unique(tables[:S])
    got = [c.get() for c in caches]
    for k in (0, 1):
        codes = [g[k].reshape(nkv, -1, 16, hd)[:, pages] for g in got]
        assert np.array_equal(codes[0], codes[1]) and np.array_equal(codes[1], codes[2])
    for k in (2, 3):
        assert np.array_equal(got[0][k][pages], got[1][k][pages]) and np.array_equal(got[1][k][pages], got[2][k][pages])

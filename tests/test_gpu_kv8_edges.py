"""The 8-bit cache's operators where they can go wrong: blocks that read as NaN, garbage
behind a sequence, malformed batches, rows and pages that are to be left alone, batches of
many sequences and of mixed lengths, odd scales and queries, caches past 32 bits, and the
operators together. Codes, scales and copies are compared exactly, attention within
test_gpu_kv8's bounds."""
import kv8_ref as ref
import numpy as np
import pytest
from test_gpu_kv8 import (E4M3, I8, NP_TYPE, Cache, attend, close, ctx, expect, ragged, tables_for,  # noqa: F401
                          tolerance, u32, zh)

pytestmark = pytest.mark.gpu


def starts_of(counts):
    return np.concatenate([[0], np.cumsum(counts)])


def agree(cache, tables, q, got, counts, lens, t, scale=None, tiled=True, odd=False):
    scale = cache.hd ** -0.5 if scale is None else scale
    want, *terms = expect(cache, tables, q, counts, lens, scale)
    close(got, want, tolerance(cache, t, want, *terms, lens, odd=odd, floor=-29 if tiled else -39))


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def fp16_pages(rng, n, nkv, hd):
    """fp16 caches of n pages of all magnitudes: blocks of zeros, subnormals, NaN, infinities."""
    x = rng.normal(size=(nkv, n, 16, hd)) * 2.0 ** rng.integers(-24, 12, (nkv, n, 1, 1))
    x = np.clip(x, -60000, 60000).astype(np.float16)
    kind = rng.integers(0, 12, (nkv, n))
    x[kind == 0] = 0
    x[kind == 1, 3, 5] = np.nan
    x[kind == 2, 15, hd - 1] = -np.inf
    x[kind == 3] = np.float16(6e-8)
    return x


def packed(x, fmt, n_tokens):
    """x [nkv][pages][16][hd] -> codes, scales [pages][nkv]; slots past n_tokens are zero."""
    x = x.astype(np.float64).copy()
    x.reshape(x.shape[0], -1, x.shape[3])[:, n_tokens:] = 0
    codes, scales = np.zeros(x.shape, np.uint8), np.zeros(x.shape[1::-1], np.float32)
    for h in range(x.shape[0]):
        for p in range(x.shape[1]):
            codes[h, p], scales[p, h] = ref.store_page(codes[h, p], 0, fmt, list(range(16)), x[h, p])
    return codes, scales


@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("n_caches,nkv,hd,n_tokens", [
    (1, 1, 64, 1), (2, 3, 128, 16), (2, 8, 64, 37), (3, 2, 128, 333), (40, 2, 64, 95), (256, 1, 64, 17), (1, 8, 128, 16000)])
def test_pack_unpack_copy(zh, ctx, fmt, n_caches, nkv, hd, n_tokens):  # noqa: F811
    rng = np.random.default_rng(n_caches * 1000 + n_tokens)
    n = -(-n_tokens // 16)
    src_n, dst_n = n + 3, 2 * n + 5
    few = min(n_caches, 3)  # (contents of their own; the other caches repeat them)
    half = [fp16_pages(rng, src_n, nkv, hd) for _ in range(few)]
    sp, dp = rng.permutation(src_n)[:n], rng.permutation(dst_n)[:n]
    old_c = rng.integers(0, 256, (nkv, dst_n, 16, hd)).astype(np.uint8)
    old_s = np.full((dst_n, nkv), 7, np.float32)
    src = zh.KvCaches([ctx.upload(half[i % few]) for i in range(n_caches)], src_n * 16, nkv, hd)
    codes, scales = ([ctx.upload(x) for _ in range(n_caches)] for x in (old_c, old_s))
    dst = zh.Kv8Caches(codes, scales, dst_n * 16, nkv, hd, fmt)
    ctx.kv8_pack_pages(dst, src, dp, sp, n_tokens)
    ctx.sync()
    want = []
    for i in range(n_caches):
        if i < few:
            c, s = old_c.copy(), old_s.copy()
            c[:, dp], s[dp] = packed(half[i][:, sp], fmt, n_tokens)
            want.append((c, s))
        c, s = want[i % few]
        assert same(scales[i].download(np.float32, s.size).reshape(s.shape), s)
        got = codes[i].download(np.uint8, c.size).reshape(c.shape)
        ok = np.ones((dst_n, nkv), bool)
        ok[dp] = np.isfinite(s[dp])
        ok = ok.T
        untouched = np.setdiff1d(np.arange(dst_n), dp)
        assert np.array_equal(got[:, untouched], c[:, untouched])
        a, b = ref.decode(got, fmt), ref.decode(c, fmt)
        for p in dp:
            assert same(a[:, p][ok[:, p]], b[:, p][ok[:, p]])
    # to other pages of another set, and within the set
    other_n = dst_n + 4
    c2, s2 = ([ctx.upload(np.zeros(x, t)) for _ in range(n_caches)] for x, t in (((nkv, other_n, 16, hd), np.uint8),
                                                                                   ((other_n, nkv), np.float32)))
    other = zh.Kv8Caches(c2, s2, other_n * 16, nkv, hd, fmt)
    to = rng.permutation(other_n)[:n]
    ctx.kv8_copy_pages(other, dst, to, dp)
    ctx.kv8_copy_pages(dst, dst, untouched[:n], dp)
    # and back to fp16: a code times its scale, rounded
    back = [ctx.upload(np.full((nkv, src_n, 16, hd), 3, np.float16)) for _ in range(n_caches)]
    ctx.kv8_unpack_pages(zh.KvCaches(back, src_n * 16, nkv, hd), other, sp, to)
    ctx.sync()
    for i in list(range(few)) + [n_caches - 1]:
        s = want[i % few][1]
        got = codes[i].download(np.uint8, old_c.size).reshape(old_c.shape)
        moved = c2[i].download(np.uint8, nkv * other_n * 16 * hd).reshape(nkv, other_n, 16, hd)
        assert np.array_equal(moved[:, to], got[:, dp]) and np.array_equal(got[:, untouched[:n]], got[:, dp])
        left = np.setdiff1d(np.arange(other_n), to)
        assert not moved[:, left].any()
        got_s, moved_s = (b[i].download(np.float32, m * nkv).reshape(m, nkv) for b, m in ((scales, dst_n), (s2, other_n)))
        assert same(moved_s[to], s[dp]) and same(got_s[untouched[:n]], s[dp]) and not moved_s[left].any()
        x = back[i].download(np.float16, nkv * src_n * 16 * hd).reshape(nkv, src_n, 16, hd)
        with np.errstate(over="ignore", invalid="ignore"):
            y = (ref.decode(moved[:, to], fmt) * s[dp].T[:, :, None, None]).astype(np.float16)
        assert same(x[:, sp], y)
        assert (x[:, np.setdiff1d(np.arange(src_n), sp)] == 3).all()


def test_pages_refused_change_nothing(zh, ctx):  # noqa: F811
    cache = Cache(ctx, np.random.default_rng(1), 5, 2, 64, I8)
    s = zh.Kv8Caches(cache.b[:2], cache.b[2:], 80, 2, 64, I8)
    with pytest.raises(zh.ZincError) as e:
        ctx.kv8_copy_pages(s, s, [1, 2], [0, 5])
    assert e.value.name == "InvalidArgument"
    ctx.sync()
    assert all(np.array_equal(a, b) for a, b in zip(cache.get(), (cache.k, cache.v, cache.ks, cache.vs)))


def test_unpack_reads_any_scale(zh, ctx):  # noqa: F811
    """Scales that are no powers of two, the range's ends, and past them (NaN)."""
    for fmt in (I8, E4M3):
        cache = Cache(ctx, np.random.default_rng(2), 12, 2, 64, fmt)
        cache.ks[:] = np.array([1 / 3, 2.0 ** -64, 2.0 ** 64, 2.0 ** -65, 2.0 ** 65, 0, -1, np.nan, np.inf, 1e-3, 7.77, 1e-30],
                               np.float32)[:, None]
        cache.put()
        out = ctx.alloc(2 * 2 * 192 * 64)
        p = np.arange(12)
        ctx.kv8_unpack_pages(zh.KvCaches([out], 192, 2, 64), zh.Kv8Caches(cache.b[:1], cache.b[2:3], 192, 2, 64, fmt), p, p)
        ctx.sync()
        got = out.download(np.float16, 2 * 192 * 64).reshape(2, 12, 16, 64)
        s = np.where([ref.usable(x) for x in cache.ks[:, 0]], cache.ks[:, 0], np.nan)
        prod = ref.decode(cache.k, fmt).reshape(2, 12, 16, 64) * s.astype(np.float64)[None, :, None, None]
        with np.errstate(over="ignore", invalid="ignore"):
            # (a code times a scale is rounded to 32 bits, then to fp16: half a step of each)
            assert same(got[:, [1, 2, 3, 4, 5, 6, 7, 8, 11]], prod.astype(np.float16)[:, [1, 2, 3, 4, 5, 6, 7, 8, 11]])
        for i in (0, 9, 10):
            close(got[:, i].astype(np.float64), prod[:, i], np.abs(prod[:, i]) * (2.0 ** -11 + 2.0 ** -23) + 2.0 ** -25)


# ---------------------------------------------------------------------------
# writes
# ---------------------------------------------------------------------------
def write(zh, ctx, kv, x, nq, nkv, hd, check=True, **more):  # noqa: F811
    """Raw rows (no norm, no rotation): k and v are quantised as they are."""
    T, size = len(x), x.itemsize
    w = (nq + 2 * nkv) * hd
    b, out = ctx.upload(x), ctx.upload(np.full((T, nq * hd), 77, x.dtype))
    t = 0 if size == 4 else 1
    f = dict(q=b, k=b, v=b, k_off=nq * hd * size, v_off=(nq + nkv) * hd * size, q_stride=w, k_stride=w, v_stride=w, type=t,
             q_out=out, pos=None, n_rows=T, n_q_heads=nq)
    f.update(more)
    ctx.qk_norm_rope_kv8_write_batched(kv, zh.QkvRows(**f))
    if check:
        ctx.sync()
    return out.download(x.dtype, T * nq * hd).reshape(T, nq * hd)


def stored(cache, tables, counts, lens, x, nq):
    """The cache after the rows x [T][nq + 2 nkv][hd]."""
    k, v, ks, vs = cache.k.copy(), cache.v.copy(), cache.ks.copy(), cache.vs.copy()
    first = 0
    for s, (c, n) in enumerate(zip(counts, lens)):
        pos = np.arange(n - c, n)
        for page in np.unique(pos // 16):
            phys, rows = tables[s, page], np.flatnonzero(pos // 16 == page)
            b = slice(phys * 16, phys * 16 + 16)
            for h in range(cache.nkv):
                for codes, scales, at in ((k, ks, nq + h), (v, vs, nq + cache.nkv + h)):
                    new = x[first + rows, at].astype(np.float64)
                    codes[h, b], scales[phys, h] = ref.store_page(codes[h, b], scales[phys, h], cache.fmt,
                                                                  list(pos[rows] % 16), new)
        first += c
    return k, v, ks, vs


def caches_agree(cache, got, want):
    for a, b in zip(got[2:], want[2:]):
        assert same(a, b)
    for a, b, s in zip(got[:2], want[:2], want[2:]):
        ok = np.repeat(np.isfinite(s).T, 16, 1)
        assert np.array_equal(ref.decode(a, cache.fmt)[ok], ref.decode(b, cache.fmt)[ok])


@pytest.mark.parametrize("decode", [True, False])
@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_write_of_no_numbers_and_of_extremes(zh, ctx, fmt, decode):  # noqa: F811
    """NaN, infinities, values past the largest scale, blocks that read as NaN already,
    scales of zero and below the least; each stays in its block."""
    rng = np.random.default_rng(11)
    counts = [1] * 24 if decode else [1, 2, 17, 3, 30, 5, 16, 4]
    lens = np.array([1 + int(rng.integers(0, 50)) + c for c in counts])
    lens[3] = counts[3]  # (its page begins anew)
    tables, total = tables_for(rng, lens, 2)
    nq, nkv, hd = 2, 2, 64
    cache = Cache(ctx, rng, total, nkv, hd, fmt)
    odd = rng.integers(0, 9, cache.ks.shape)
    for v, x in ((0, np.nan), (1, np.inf), (2, 0), (3, 2.0 ** -70), (4, -1), (5, 2.0 ** 64)):
        cache.ks[odd == v] = x
    cache.put()
    T = sum(counts)
    x = (rng.normal(size=(T, nq + 2 * nkv, hd)) * 2.0 ** rng.integers(-40, 40, (T, 1, 1))).astype(np.float32)
    x[rng.integers(0, T, 3), nq, 5] = np.nan
    x[rng.integers(0, T, 3), nq + 1, 63] = np.inf
    x[rng.integers(0, T, 3), nq + 2, 0] = -np.inf
    x[rng.integers(0, T, 2), nq + 3, 9] = 3e38
    x[rng.integers(0, T, 3), nq + 3] = 0
    x[0, nq] = 2.0 ** -149
    kv = cache.batch(zh, tables, lens, None if decode else starts_of(counts))
    out = write(zh, ctx, kv, x, nq, nkv, hd)
    assert np.array_equal(out, x[:, :nq].reshape(T, -1))
    caches_agree(cache, cache.get(), stored(cache, tables, counts, lens, x, nq))


@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_write_malformed_batches(zh, ctx, fmt):  # noqa: F811
    """What has no place is left out and reported; the rest is written."""
    rng = np.random.default_rng(12)
    nq, nkv, hd = 1, 1, 64

    def go(tables, lens, starts, T, total):
        cache = Cache(ctx, rng, total, nkv, hd, fmt)
        x = rng.normal(size=(T, 3, hd)).astype(np.float32)
        with pytest.raises(zh.ZincError) as e:
            write(zh, ctx, cache.batch(zh, u32(tables), lens, starts), x, nq, nkv, hd)
        assert e.value.name == "InvalidArgument"
        ctx.sync()  # (reported once)
        return cache, x

    # a page outside the cache: the sequence's other pages are written
    tables = np.array([[0, 99, 2], [3, 4, 5]])
    cache, x = go(tables, [40, 20], [0, 40, 45], 45, 6)
    t2, c2 = tables.copy(), Cache.__new__(Cache)
    c2.__dict__.update(cache.__dict__)
    for a in ("k", "v"):  # (a place for what is left out)
        setattr(c2, a, np.concatenate([getattr(cache, a), np.zeros((nkv, 16, hd), np.uint8)], 1))
        setattr(c2, a + "s", np.concatenate([getattr(cache, a + "s"), np.ones((1, nkv), np.float32)]))
    t2[0, 1] = 6
    want = stored(c2, t2, [40, 5], [40, 20], x, nq)
    caches_agree(cache, cache.get(), [want[0][:, :96], want[1][:, :96], want[2][:6], want[3][:6]])
    # more rows than tokens: the last ones are written
    cache, x = go([[0, 1], [2, 3]], [5, 20], [0, 9, 12], 12, 4)
    caches_agree(cache, cache.get(), stored(cache, u32([[0, 1], [2, 3]]), [5, 3], [5, 20], x[4:], nq))
    # a length past the table
    cache, x = go([[0, 1], [2, 3]], [40, 20], [0, 10, 13], 13, 4)
    caches_agree(cache, cache.get(), stored(cache, u32([[0, 1], [2, 3]]), [2, 3], [32, 20], x[[0, 1, 10, 11, 12]], nq))
    # rows that fall, and that pass the call's: nothing out of place
    for starts in ([0, 9, 5], [0, 3, 1 << 31], [7, 3, 6]):
        cache, x = go([[0, 1], [2, 3]], [20, 20], starts, 6, 4)


@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_write_leaves_other_rows_and_pages(zh, ctx, fmt):  # noqa: F811
    rng = np.random.default_rng(13)
    lens, tables = [20, 0, 33], u32([[5, 1, 9], [77, 77, 77], [2, 7, 0]])
    nq, nkv, hd = 2, 1, 128
    cache = Cache(ctx, rng, 10, nkv, hd, fmt)
    x = rng.normal(size=(12, 4, hd)).astype(np.float16)
    out = write(zh, ctx, cache.batch(zh, tables, lens, [2, 5, 5, 9]), x, nq, nkv, hd)  # (rows 0, 1 and 9 .. are of none)
    assert (out[[0, 1, 9, 10, 11]] == 77).all() and np.array_equal(out[2:9], x[2:9, :2].reshape(7, -1))
    caches_agree(cache, cache.get(), stored(cache, tables, [3, 0, 4], lens, x[2:9], nq))
    cache = Cache(ctx, rng, 10, nkv, hd, fmt)
    out = write(zh, ctx, cache.batch(zh, tables, lens), x[:3], nq, nkv, hd)  # (a row a sequence, the second has no tokens)
    assert (out[1] == 77).all()
    caches_agree(cache, cache.get(), stored(cache, tables, [1, 0, 1], lens, x[[0, 2]], nq))


@pytest.mark.parametrize("fmt", [I8, E4M3])
def test_write_one_row_at_a_time_and_all_at_once(zh, ctx, fmt):  # noqa: F811
    """Rows written a step each, over growing scales, and in one call: equal scales, values
    within what rounding again costs."""
    rng = np.random.default_rng(14)
    nq, nkv, hd, n = 2, 2, 64, 40
    x = rng.normal(size=(n, 6, hd)).astype(np.float32)
    tables = u32([[2, 0, 1]])
    one, all_ = Cache(ctx, rng, 3, nkv, hd, fmt), Cache(ctx, rng, 3, nkv, hd, fmt)
    for i in range(n):
        write(zh, ctx, one.batch(zh, tables, [i + 1]), x[i:i + 1], nq, nkv, hd, check=False)
    write(zh, ctx, all_.batch(zh, tables, [n], [0, n]), x, nq, nkv, hd)
    a, b = one.get(), all_.get()
    for i in (2, 3):
        assert np.array_equal(a[i], b[i])  # (a scale depends on the largest value only)
    for c, s, at in ((0, 2, 2), (1, 3, 4)):
        for h in range(nkv):
            for g in (a, b):
                got = np.stack([ref.decode(g[c][h, tables[0, p // 16] * 16 + p % 16], fmt) * g[s][tables[0, p // 16], h]
                                for p in range(n)])
                sc = np.array([g[s][tables[0, p // 16], h] for p in range(n)])[:, None]
                v = x[:, at + h].astype(np.float64)
                # each rise rounds once more, at scales up to the last: half a step, and its halves
                # (e4m3: a value's own rounding, and those below the normal range)
                step = 0.5 * sc if fmt == I8 else np.maximum(np.abs(v) * 2.0 ** -4, 2.0 ** -10 * sc)
                assert (np.abs(got - v) <= 3.01 * step).all()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
MIXED = [  # counts, lens, heads per kv head, kv heads, head_dim
    ([1] * 9 + [200], [700] * 9 + [900], 4, 2, 64),                 # streamed rows and LDS tiles in one call
    ([40, 1, 3, 300, 1, 60, 9, 1, 1, 130], None, 2, 2, 128),
    ([1, 1, 150], [3000, 17, 160], 4, 1, 128),                      # few sequences: all on tiles
    ([150] + [0] * 5 + [1] * 70, None, 2, 1, 64),                   # more than 64 sequences
    ([140, 0, 1] * 30, None, 1, 1, 64),
    ([11] * 20, None, 3, 1, 128),                                   # tiles of 32 that cut a row's heads
    ([5] * 9, [2000] * 9, 71, 1, 64),
    ([50, 1] * 5 + [200], [2500, 1300] * 5 + [1700], 2, 1, 64),     # row tiles in shares, and LDS tiles
    ([20, 3, 40] * 14, [2500, 77, 640] * 14, 2, 1, 64),
    ([1] * 90, [1800, 900, 2500] * 30, 4, 2, 128),
]


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("case", MIXED, ids=lambda c: str(len(c[0])) + "x" + str(max(c[0])))
def test_mixed_batches(zh, ctx, t, case):  # noqa: F811
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + G)
    lens = ragged(rng, counts, lens)
    lens[np.array(counts) == 0] = 25
    tables, total = tables_for(rng, lens, 2)
    cache = Cache(ctx, rng, total, nkv, hd, (I8, E4M3)[sum(counts) % 2])
    q, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts_of(counts))
    agree(cache, tables, q, got, counts, lens, t)


SHAPES = [  # streamed, in one workgroup a sequence and in shares; LDS tiles whole and cut
    ([1, 2, 1], [40, 33, 200], 4, 2, 64),
    ([1, 1, 1], [3000, 900, 2100], 4, 2, 128),
    ([40, 7], [60, 300], 3, 1, 128),
    ([260, 3], [700, 300], 1, 2, 64),
    ([300], [4000], 1, 1, 128),
    ([40, 7], [2600, 300], 3, 1, 128),
    ([60, 1, 20], [1500, 3000, 2200], 2, 1, 64),
]


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: str(len(c[0])) + "x" + str(max(c[0])))
def test_garbage_around_the_tokens(zh, ctx, case, fmt, t):  # noqa: F811
    """NaN codes behind the last token, NaN scales of every other page, table entries past
    the sequence's pages anywhere; scales that are no powers of two; rows with room
    between them, in place of q; other rows and the room left as they were; the same again bit for bit."""
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts))
    tables, total = tables_for(rng, lens, 5)
    cache = Cache(ctx, rng, total, nkv, hd, fmt, odd_scales=True, spread=3)
    seen = np.zeros(total * 16, bool)
    for s, n in enumerate(lens):
        p = np.arange(n)
        seen[tables[s, p // 16].astype(np.int64) * 16 + p % 16] = True
    for c in (cache.k, cache.v):
        c[:, ~seen] = 0x7F if fmt == E4M3 else 0x80
    used = seen.reshape(-1, 16).any(1)
    for x in (cache.ks, cache.vs):
        x[~used] = np.nan
    cache.put()
    wide = np.concatenate([tables, np.full((len(lens), 3), 0xFFFFFFFF, np.uint32)], 1)
    for s, n in enumerate(lens):
        wide[s, -(-n // 16):] = 0xFFFFFFF0
    T, nh, first = sum(counts), G * nkv, 2
    w, room = nh * hd, nh * hd + 32
    rows = T + 5
    x = rng.normal(size=(rows, room)).astype(NP_TYPE[t])
    starts = first + starts_of(counts)
    kv = cache.batch(zh, wide, lens, starts)
    most, longest = max(counts) + 2, max(lens) + 9
    ws = ctx.alloc(ctx.flash_attn_kv8_ws(kv, nh, rows, most, longest))
    runs = []
    for _ in range(2):
        b = ctx.upload(x)
        ctx.flash_attn_kv8(kv, zh.AttnRows(q=b, out=b, ws=ws, n_rows=rows, max_rows=most, max_len=longest, n_heads=nh, type=t,
                                           q_stride=room, out_stride=room))
        ctx.sync()
        runs.append(b.download(x.dtype, x.size).reshape(x.shape))
    assert np.array_equal(runs[0], runs[1])
    got = runs[0]
    assert np.array_equal(got[:, w:], x[:, w:])
    assert np.array_equal(got[:first], x[:first]) and np.array_equal(got[first + T:], x[first + T:])
    q = x[first:first + T, :w].reshape(T, nh, hd)
    out = got[first:first + T, :w].reshape(T, nh, hd).astype(np.float64)
    cache.ks[~used] = cache.vs[~used] = 1
    agree(cache, tables, q, out, counts, lens, t, odd=True)


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: str(len(c[0])) + "x" + str(max(c[0])))
def test_blocks_that_read_as_nan(zh, ctx, case, t):  # noqa: F811
    """Rows that see one are NaN in that kv head, all others as without."""
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + 1)
    tables, total = tables_for(rng, lens, 1)
    cache = Cache(ctx, rng, total, nkv, hd, I8)
    starts = starts_of(counts)
    s = len(counts) - 1
    page = (lens[s] - counts[s]) // 16 + (1 if counts[s] > 40 else 0)  # (the rows' own, or one that some see)
    q = rng.normal(size=(sum(counts), G * nkv, hd)).astype(NP_TYPE[t])
    want, *terms = expect(cache, tables, q, counts, lens, hd ** -0.5)
    tol = tolerance(cache, t, want, *terms, lens, floor=-29)
    for x, value in ((cache.ks, np.nan), (cache.vs, 2.0 ** 65), (cache.ks, 0)):
        keep = x.copy()
        x[tables[s, page], 0] = value
        cache.put()
        _, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts, q=q)
        x[:] = keep
        row = np.arange(counts[s])
        sees = lens[s] - counts[s] + row + 1 > 16 * page
        hit = np.zeros(got.shape, bool)
        hit[starts[s] + row[sees], :G] = True
        assert hit.any() and np.isnan(got[hit]).all()
        close(got[~hit], want[~hit], tol[~hit])


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: str(len(c[0])) + "x" + str(max(c[0])))
def test_queries_and_scales_of_any_size(zh, ctx, case, t):  # noqa: F811
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + 2)
    tables, total = tables_for(rng, lens, 1)
    cache = Cache(ctx, rng, total, nkv, hd, E4M3, spread=2)
    starts = starts_of(counts)
    go = lambda **k: attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts, **k)  # noqa: E731
    q, base = go(scale=0.5)
    near, *terms = expect(cache, tables, q, counts, lens, 0.5)
    tol = tolerance(cache, t, near, *terms, lens, floor=-29)
    close(base, near, tol)
    _, got = go(scale=-0.5, q=q)
    agree(cache, tables, q, got, counts, lens, t, -0.5)
    if t == 0:  # (f32 q of any size: the products' exponents only)
        for e in (60, -60, 100, -100):
            _, got = go(scale=2.0 ** (-1 - e), q=np.ldexp(q, e))
            assert np.array_equal(got, base)
    _, got = go(scale=1e-38, q=q)  # (flat)
    agree(cache, tables, q, got, counts, lens, t, 1e-38)
    _, got = go(q=np.zeros_like(q))
    agree(cache, tables, np.zeros_like(q), got, counts, lens, t)
    # all of the weight on the largest score, where it passes the next by a hundredth
    first = 0
    want, sure = np.zeros(got.shape), np.zeros(got.shape, bool)
    for s, (c, n) in enumerate(zip(counts, lens)):
        p = np.arange(n)
        at = tables[s, p // 16].astype(np.int64) * 16 + p % 16
        for h in range(nkv):
            k = ref.decode(cache.k[h, at], E4M3) * cache.ks[at // 16, h][:, None]
            v = ref.decode(cache.v[h, at], E4M3) * cache.vs[at // 16, h][:, None]
            for i in range(c):
                x = q[first + i, h * G:(h + 1) * G].astype(np.float64) @ k[:n - c + i + 1].T
                top = np.sort(x, 1)
                want[first + i, h * G:(h + 1) * G] = v[x.argmax(1)]
                if x.shape[1] > 1:
                    sure[first + i, h * G:(h + 1) * G] = (top[:, -1] - top[:, -2] > 0.01 * np.abs(x).max(1))[:, None]
        first += c
    assert sure.any()
    tol1 = np.abs(want[sure]) * 2.0 ** (-11 if t else -20) + (2.0 ** -25 if t else 0)
    for scale in (1e6, 3e6, 1e7, 3e7, 1e8, 1e12, 1e30):
        _, got = go(scale=scale, q=q)
        close(got[sure], want[sure], tol1)
    _, got = go(scale=3e38, q=q)  # (scores past the range of 32 bits: that, or no number)
    ok = ~np.isnan(got[sure])
    close(got[sure][ok], want[sure][ok], tol1[ok])
    # rows of infinities and NaN stay by themselves
    q[1, 0, 5], q[-1, -1, 0] = np.nan, np.inf
    _, got = go(scale=0.5, q=q)
    hit = np.zeros(got.shape, bool)
    hit[1, 0] = hit[-1, -1] = True
    assert not np.isfinite(got[hit]).any()
    close(got[~hit], near[~hit], tol[~hit])


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("case", SHAPES, ids=lambda c: str(len(c[0])) + "x" + str(max(c[0])))
def test_attention_of_malformed_batches(zh, ctx, case, t):  # noqa: F811
    """Reported once by the next sync; what is defined is right, the rest of out left alone."""
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + 3)
    tables, total = tables_for(rng, lens, 1)
    cache = Cache(ctx, rng, total, nkv, hd, I8)
    starts = starts_of(counts)

    def run(**k):
        f = dict(tables=tables, lens=lens, starts=starts)
        f.update({n: k.pop(n) for n in list(k) if n in f})
        q, got = attend(zh, ctx, rng, cache, f["tables"], counts, f["lens"], G, t, f["starts"], check=False, **k)
        with pytest.raises(zh.ZincError) as e:
            ctx.sync()
        assert e.value.name == "InvalidArgument"
        ctx.sync()
        return q, got

    # a page outside reads as page 0
    wrong, zero = tables.copy(), tables.copy()
    wrong[-1, 0], zero[-1, 0] = total, 0
    q, got = run(tables=wrong)
    agree(cache, zero, q, got, counts, lens, t)
    # lengths past max_len are cut there
    cut = max(lens) - 5
    q, got = run(max_len=cut)
    want, *terms = expect_cut(cache, tables, q, counts, lens, cut)
    close(got, want, tolerance(cache, t, want, *terms, lens, floor=-29))
    # rows past max_rows are left as they were
    if max(counts) > 1:
        most = max(counts) - 1
        q, got = run(max_rows=most)
        left = np.concatenate([np.arange(c) >= most for c in counts])
        assert (got[left] == 77).all()
        want, *terms = expect(cache, tables, q, counts, lens, hd ** -0.5)
        tol = tolerance(cache, t, want, *terms, lens, floor=-29)
        close(got[~left], want[~left], tol[~left])
    # rows that fall or pass the call's, more rows than tokens
    T = sum(counts)
    for starts_bad in ([T] + [0] * len(counts), [0] * len(counts) + [T + 9], [0] * len(counts) + [0xFFFFFFFF]):
        run(starts=u32(starts_bad))
    run(lens=[0] * len(counts) if max(counts) == 1 else [1] * len(counts), max_len=max(lens))


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("G", [4, 80])
def test_sequences_without_rows(zh, ctx, G, t):  # noqa: F811
    """Their lengths and pages may be anything, in a write and in attention, in both ways to
    say whose the rows are."""
    rng = np.random.default_rng(G)
    counts, lens, hd, nkv = [2, 0, 3, 0, 0], [50, 1 << 31, 900, 0xFFFFFFFF, 7], 64, 1
    live = [n if c else 0 for c, n in zip(counts, lens)]
    tables, total = tables_for(rng, live, 1)
    tables[1] = tables[3:] = 0xFFFFFF00
    cache = Cache(ctx, rng, total, nkv, hd, E4M3)
    kv = cache.batch(zh, tables, lens, starts_of(counts))
    nq = 2
    x = rng.normal(size=(5, nq + 2 * nkv, hd)).astype(np.float32)
    write(zh, ctx, kv, x, nq, nkv, hd)
    cache.k, cache.v, cache.ks, cache.vs = stored(cache, tables, counts, live, x, nq)
    caches_agree(cache, cache.get(), (cache.k, cache.v, cache.ks, cache.vs))
    cache.put()
    q, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts_of(counts), max_len=912)
    agree(cache, tables, q, got, counts, live, t)
    # a row a sequence, fewer rows than sequences
    order = [0, 2, 1, 3, 4]
    q, got = attend(zh, ctx, rng, cache, tables[order], [1, 1], u32(lens)[order], G, t, None, max_len=912)
    agree(cache, tables[order], q, got, [1, 1], [live[i] for i in order[:2]], t)


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("counts,lens,G", [([1, 1, 1], [40, 700, 2600], 4), ([3, 50, 9], [3, 400, 77], 4), ([90, 1], [300, 20], 4)])
def test_stacked_rows_in_place(zh, ctx, t, counts, lens, G):  # noqa: F811
    """Rows q | k | v | room of one buffer: q rotated in place, its result in the room; k and v
    as they were."""
    rng = np.random.default_rng(sum(lens))
    nkv, hd = 2, 64
    nq, T = G * nkv, sum(counts)
    tables, total = tables_for(rng, lens, 1)
    cache = Cache(ctx, rng, total, nkv, hd, (I8, E4M3)[t])
    cache.ks[:] = cache.vs[:] = 2.0 ** -5
    cache.put()
    kv = cache.batch(zh, tables, lens, None if max(counts) == 1 else starts_of(counts))
    w, W = (nq + 2 * nkv) * hd, (2 * nq + 2 * nkv) * hd + 16
    x = rng.normal(size=(T, W)).astype(NP_TYPE[t])
    b, size = ctx.upload(x), x.itemsize
    freq = (1e4 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    same_rows = dict(q_stride=W, k_stride=W, v_stride=W, q_out_stride=W)
    ctx.qk_norm_rope_kv8_write_batched(kv, zh.QkvRows(q=b, k=b, v=b, q_out=b, k_off=nq * hd * size,
                                                      v_off=(nq + nkv) * hd * size, type=t, pos=None, n_rows=T,
                                                      n_q_heads=nq, inv_freq=ctx.upload(freq), rope_dim=hd, **same_rows))
    ws = ctx.alloc(ctx.flash_attn_kv8_ws(kv, nq, T, max(counts), max(lens)))
    ctx.flash_attn_kv8(kv, zh.AttnRows(q=b, out=b, out_off=w * size, q_stride=W, out_stride=W, ws=ws, n_rows=T, type=t,
                                       max_rows=max(counts), max_len=max(lens), n_heads=nq))
    ctx.sync()
    got = b.download(x.dtype, x.size).reshape(x.shape)
    pos = np.concatenate([np.arange(n - c, n) for n, c in zip(lens, counts)])
    h = x[:, :w].reshape(T, nq + 2 * nkv, hd)
    turned = ref.turned(h[:, :nq + nkv], None, freq, pos, 1e-6, hd)
    q = got[:, :nq * hd].reshape(T, nq, hd)
    mag = np.abs(h[:, :nq]).astype(np.float64)
    mag = np.concatenate([mag[..., :hd // 2] + mag[..., hd // 2:]] * 2, -1)
    close(q.astype(np.float64), turned[:, :nq], 2.0 ** -19 * mag + np.abs(turned[:, :nq]) * 2.0 ** (-11 if t else -24) +
          (2.0 ** -25 if t else 0))
    assert np.array_equal(got[:, nq * hd:w], x[:, nq * hd:w]) and np.array_equal(got[:, W - 16:], x[:, W - 16:])
    y = h.astype(np.float64)
    y[:, nq:nq + nkv] = turned[:, nq:]
    cache.k, cache.v, cache.ks, cache.vs = stored(cache, tables, counts, lens, y, nq)
    caches_agree(cache, cache.get(), (cache.k, cache.v, cache.ks, cache.vs))
    agree(cache, tables, q, got[:, w:w + nq * hd].reshape(q.shape).astype(np.float64), counts, lens, t)


def expect_cut(cache, tables, q, counts, lens, cut):
    """The rows see the tokens below `cut` only."""
    parts, first = [], 0
    for s, (c, n) in enumerate(zip(counts, lens)):
        rows = []
        for i in range(c):
            m = min(n - c + i + 1, cut)
            rows.append(ref.attention(q[first + i:first + i + 1], cache.k, cache.v, cache.ks, cache.vs, tables[s], 1, m,
                                      cache.hd ** -0.5, cache.fmt))
        parts += rows
        first += c
    return [np.concatenate([p[i] for p in parts]) for i in range(4)]


def test_two_contexts_at_once(zh, ctx):  # noqa: F811
    """Calls that overlap, with a workspace each; the results are those of each alone."""
    rng = np.random.default_rng(31)
    other = zh.Context(0)
    try:
        work = []
        for c, (counts, lens, G, nkv, hd) in ((ctx, SHAPES[1]), (other, SHAPES[4]), (ctx, SHAPES[3]), (other, SHAPES[1])):
            tables, total = tables_for(rng, lens, 1)
            cache = Cache(c, rng, total, nkv, hd, E4M3)
            T, nh = sum(counts), G * nkv
            q = rng.normal(size=(T, nh, hd)).astype(np.float32)
            kv = cache.batch(zh, tables, lens, starts_of(counts))
            out = c.alloc(q.nbytes)
            rows = zh.AttnRows(q=c.upload(q), out=out, n_rows=T, max_rows=max(counts), max_len=max(lens), n_heads=nh,
                               ws=c.alloc(c.flash_attn_kv8_ws(kv, nh, T, max(counts), max(lens))))
            work.append((c, kv, rows, out, q.size))
        alone = []
        for c, kv, rows, out, n in work:
            c.flash_attn_kv8(kv, rows)
            c.sync()
            alone.append(out.download(np.float32, n))
        for _ in range(20):
            for c, kv, rows, out, n in work:
                c.flash_attn_kv8(kv, rows)
        for (c, kv, rows, out, n), a in zip(work, alone):
            c.sync()
            assert np.array_equal(out.download(np.float32, n), a)
    finally:
        other.close()


@pytest.mark.parametrize("fmt,t", [(I8, 0), (E4M3, 1)])
def test_a_prompt_forked_drafted_and_read_back(zh, ctx, fmt, t):  # noqa: F811
    """A prompt's fp16 pages packed, two children that share them, a page of each copied
    before its own rows are written, a chunk and drafted tokens in one batch, decode steps,
    and the cache read back: every step against the plain operators."""
    rng = np.random.default_rng(41)
    nkv, G, hd, P, prompt = 2, 4, 128, 64, 75
    nq = G * nkv
    pool = zh.KvPagePool(P, 16)
    pool.alloc_pages(1, 5)
    half = (rng.normal(size=(nkv, 8, 16, hd))).astype(np.float16)
    hb = ctx.upload(half)
    cache = Cache(ctx, rng, P, nkv, hd, fmt)
    ks, vs = (zh.Kv8Caches([cache.b[i]], [cache.b[i + 2]], P * 16, nkv, hd, fmt) for i in (0, 1))
    pages = pool.pages(1)
    src = rng.permutation(8)[:5]
    for dst, codes, scales in ((ks, cache.k, cache.ks), (vs, cache.v, cache.vs)):
        ctx.kv8_pack_pages(dst, zh.KvCaches([hb], 128, nkv, hd), pages, src, prompt)
        c, s = packed(half[:, src], fmt, prompt)
        codes.reshape(nkv, P, 16, hd)[:, pages] = c
        scales[pages] = s
    lens = {1: prompt}
    for child in (2, 3):
        pool.fork(1, child, 5)
        a, b = pool.unshare(child, 4)
        for x, codes, scales in ((ks, cache.k, cache.ks), (vs, cache.v, cache.vs)):
            ctx.kv8_copy_pages(x, x, [b], [a])
            codes.reshape(nkv, P, 16, hd)[:, b] = codes.reshape(nkv, P, 16, hd)[:, a]
            scales[b] = scales[a]
        lens[child] = prompt
    ctx.sync()
    freq = (1e4 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    wk = (1 + 0.1 * rng.normal(size=hd)).astype(np.float32)
    F, WK = ctx.upload(freq), ctx.upload(wk)
    for counts in ((33, 5, 1), (1, 1, 1), (2, 0, 7), (1, 1, 1)):
        for s, c in zip((1, 2, 3), counts):
            lens[s] += c
            need = -(-lens[s] // 16) - len(pool.pages(s))
            if need > 0:
                pool.alloc_pages(s, need)
        tables = np.zeros((3, 12), np.uint32)
        for i in range(3):
            p = pool.pages(i + 1)
            tables[i, :len(p)] = p
        L, T = [lens[s] for s in (1, 2, 3)], sum(counts)
        kv = cache.batch(zh, tables, L, None if set(counts) == {1} else starts_of(counts))
        x = rng.normal(size=(T, nq + 2 * nkv, hd)).astype(NP_TYPE[t])
        qo = ctx.alloc(x.itemsize * T * nq * hd)
        q = write(zh, ctx, kv, x, nq, nkv, hd, q_out=qo, inv_freq=F, rope_dim=hd, q_norm_w=WK, k_norm_w=WK)
        q = qo.download(NP_TYPE[t], T * nq * hd).reshape(T, nq, hd)
        pos = np.concatenate([np.arange(n - c, n) for n, c in zip(L, counts)])
        y = x.astype(np.float64)
        y[:, nq:nq + nkv] = ref.turned(x[:, nq:nq + nkv], wk, freq, pos, 1e-6, hd)
        cache.k, cache.v, cache.ks, cache.vs = stored(cache, tables, counts, L, y, nq)
        caches_agree(cache, cache.get(), (cache.k, cache.v, cache.ks, cache.vs))
        out = ctx.alloc(q.nbytes)
        ctx.flash_attn_kv8(kv, zh.AttnRows(q=qo, out=out, n_rows=T, max_rows=max(counts), max_len=max(L), n_heads=nq, type=t,
                                           ws=ctx.alloc(ctx.flash_attn_kv8_ws(kv, nq, T, max(counts), max(L)))))
        ctx.sync()
        got = out.download(NP_TYPE[t], T * nq * hd).reshape(q.shape).astype(np.float64)
        agree(cache, tables, q, got, counts, L, t)
    pages = pool.pages(3)
    back = ctx.alloc(2 * nkv * 12 * 16 * hd)
    ctx.kv8_unpack_pages(zh.KvCaches([back], 192, nkv, hd), vs, np.arange(len(pages)), pages)
    ctx.sync()
    got = back.download(np.float16, nkv * 192 * hd).reshape(nkv, 12, 16, hd)[:, :len(pages)]
    want = ref.decode(cache.v.reshape(nkv, P, 16, hd)[:, pages], fmt) * cache.vs[pages].T[:, :, None, None]
    assert np.array_equal(got, want.astype(np.float16))


def test_caches_past_32_bits(zh, ctx):  # noqa: F811
    """4 GiB of codes each: rows written to the last pages, attended there and, copied,
    in low ones; packed and read back there."""
    rng = np.random.default_rng(51)
    nkv, G, hd, tokens = 4, 4, 128, (1 << 23) + 4096
    last, fmt, nh = tokens // 16, I8, 16
    size = nkv * tokens * hd
    assert size > 1 << 32
    bufs = [ctx.alloc(size), ctx.alloc(size), ctx.alloc(size // hd // 4), ctx.alloc(size // hd // 4)]
    lens, counts = [700, 90], [700, 90]
    near = np.zeros((2, 44), np.uint32)
    near[0], near[1, :6] = np.arange(44), np.arange(44, 50)
    far = (last - 1 - near).astype(np.uint32)
    x = rng.normal(size=(790, nh + 2 * nkv, hd)).astype(np.float16)
    small = Cache(ctx, rng, 50, nkv, hd, fmt)
    want = stored(small, near, counts, lens, x, nh)
    small.k, small.v, small.ks, small.vs = want
    batch = lambda t: zh.Kv8Batch(*bufs, ctx.upload(t), ctx.upload(u32(lens)), row_start=ctx.upload(u32([0, 700, 790])),  # noqa: E731
                                  n_seq=2, table_stride=44, cache_tokens=tokens, n_kv_heads=nkv, head_dim=hd, type=fmt)
    write(zh, ctx, batch(far), x, nh, nkv, hd)
    s = zh.Kv8Caches(bufs[:2], bufs[2:], tokens, nkv, hd, fmt)
    p = np.arange(50)
    run = []
    for t, rows in ((0, 790), (1, 790)):
        q = rng.normal(size=(rows, nh, hd)).astype(NP_TYPE[t])
        for where in (far, near):
            if where is near:
                ctx.kv8_copy_pages(s, s, p, last - 1 - p)
            kv = batch(where)
            out = ctx.alloc(q.nbytes)
            ctx.flash_attn_kv8(kv, zh.AttnRows(q=ctx.upload(q), out=out, n_rows=rows, max_rows=700, max_len=700, n_heads=nh,
                                               type=t, ws=ctx.alloc(ctx.flash_attn_kv8_ws(kv, nh, rows, 700, 700))))
            ctx.sync()
            run.append(out.download(NP_TYPE[t], q.size).reshape(q.shape))
        assert np.array_equal(run[-2], run[-1])
        only = [0, 1, 300, 699]
        for i in only:
            w, *terms = ref.attention(q[i:i + 1], small.k, small.v, small.ks, small.vs, near[0], 1, i + 1, hd ** -0.5, fmt)
            close(run[-1][i:i + 1].astype(np.float64), w, tolerance(small, t, w, *terms, [700], floor=-29))
    # one row a sequence, streamed
    lens1 = u32([700, 90])
    outs = []
    q = rng.normal(size=(2, nh, hd)).astype(np.float32)
    for where in (far, near):
        kv = zh.Kv8Batch(*bufs, ctx.upload(where), ctx.upload(lens1), n_seq=2, table_stride=44, cache_tokens=tokens,
                         n_kv_heads=nkv, head_dim=hd, type=fmt)
        out = ctx.alloc(q.nbytes)
        ctx.flash_attn_kv8(kv, zh.AttnRows(q=ctx.upload(q), out=out, n_rows=2, max_rows=1, max_len=700, n_heads=nh,
                                           ws=ctx.alloc(ctx.flash_attn_kv8_ws(kv, nh, 2, 1, 700))))
        ctx.sync()
        outs.append(out.download(np.float32, q.size).reshape(q.shape))
    assert np.array_equal(*outs)
    agree(small, near, q, outs[0].astype(np.float64), [1, 1], lens, 0)
    # the far pages read back and packed again
    half = [ctx.alloc(2 * nkv * 50 * 16 * hd) for _ in range(2)]
    h = zh.KvCaches(half, 800, nkv, hd)
    ctx.kv8_unpack_pages(h, s, p, last - 1 - p)
    ctx.kv8_pack_pages(s, h, last - 60 - p, p, 790)
    ctx.sync()
    for i, (c, sc) in enumerate(((small.k, small.ks), (small.v, small.vs))):
        y = (ref.decode(c, fmt).reshape(nkv, 50, 16, hd) * sc.T[:, :, None, None]).astype(np.float16)
        assert np.array_equal(half[i].download(np.float16, y.size).reshape(y.shape), y)
        pc, ps = packed(y, fmt, 790)
        got_s = bufs[2 + i].download(np.float32, nkv * 50, (last - 60 - 49) * nkv * 4).reshape(50, nkv)[::-1]
        assert np.array_equal(got_s, ps)
        for hh in range(nkv):
            got = bufs[i].download(np.uint8, 50 * 16 * hd, (hh * tokens + (last - 60 - 49) * 16) * hd).reshape(50, 16, hd)[::-1]
            assert np.array_equal(got, pc[hh])


def test_write_of_more_pages_than_a_launch_has(zh, ctx):  # noqa: F811
    """2250 workgroups a page, 2^23 a launch: 3800 pages take two."""
    rng = np.random.default_rng(61)
    H, hd, S = 2000, 64, 3800
    base = rng.normal(size=(16, H, hd)).astype(np.float16)
    x = ctx.upload(base[np.arange(S) % 16])
    pages = rng.permutation(S).astype(np.uint32)
    size = S * 16 * H * hd
    bufs = [ctx.alloc(size), ctx.alloc(size), ctx.alloc(4 * S * H), ctx.alloc(4 * S * H)]
    kv = zh.Kv8Batch(*bufs, ctx.upload(pages), ctx.upload(np.ones(S, np.uint32)), row_start=ctx.upload(u32(np.arange(S + 1))),
                     n_seq=S, table_stride=1, cache_tokens=16 * S, n_kv_heads=H, head_dim=hd, type=I8)
    out = ctx.alloc(2 * S * H * hd)
    ctx.qk_norm_rope_kv8_write_batched(kv, zh.QkvRows(q=x, k=x, v=x, type=1, q_out=out, pos=None, n_rows=S, n_q_heads=H))
    ctx.sync()
    got = out.download(np.float16, S * H * hd).reshape(S, H, hd)
    assert np.array_equal(got[[0, 3727, 3728, S - 1]], base[[0, 3727 % 16, 3728 % 16, (S - 1) % 16]])
    scales = [bufs[i].download(np.float32, S * H).reshape(S, H) for i in (2, 3)]
    for s in (0, 1, 3726, 3727, 3728, 3729, S - 1):
        for h in (0, 1, 999, H - 1):
            c, want = ref.store_page(np.zeros((16, hd), np.uint8), 0, I8, [0], base[s % 16, h:h + 1].astype(np.float64))
            for i in (0, 1):
                assert scales[i][pages[s], h] == want
                codes = bufs[i].download(np.uint8, 16 * hd, ((h * S + int(pages[s])) * 16) * hd).reshape(16, hd)
                assert np.array_equal(codes, c)

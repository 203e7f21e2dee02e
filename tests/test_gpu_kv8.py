"""The paged KV cache in 8 bits on the GPU, against plain numpy in 64 bits.

Tolerances. Codes and scales: none. k goes from the row to its code in 64 bits, a
value within 2^-45 of the border of two codes is not met by chance.
  q: as test_gpu_kv_batch's rope, 2^-19 (|a| + |b|) of a pair and the store's
    rounding.
  attention: as test_gpu_kv_batch's (q and weights in two pieces, 22 bits): a score
    is off by at most 2^-18 A, A = 1.45 scale sum |q_i k_i| of the row's largest,
    and a weight by as much and 2^-21; sums over n tokens add n / 32 + 64 steps of
    2^-23. Here the block's exponent E = |log2 b| is added to the score, 2^-23 (A + E)
    more, and a scale that is no power of two adds 2^-20 (its exponent's fraction,
    its reciprocal): |error| <= W (2^-17 A + (n / 32 + 84 + 2 E) 2^-23 [+ 2^-19]),
    W = sum w |v|. Pieces of weights end at fp16's least subnormal, 2^-24: a weight is
    off by 2^-25 where the row's largest w b is 2^14 (on LDS tiles 2^4 at least),
    which adds 2^-39 (2^-29) max(w b) sum |Vc|. ZH_F16 adds 2^-11 W where the
    weights are one piece, and the store's rounding.
"""
import kv8_ref as ref
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
I8, E4M3 = ref.I8, ref.E4M3
NP_TYPE = {0: np.float32, 1: np.float16}


@pytest.fixture(scope="module")
def zh():
    import zinc_amd
    return zinc_amd


@pytest.fixture()
def ctx(zh):
    c = zh.Context(0)
    yield c
    c.close()


def u32(x):
    return np.ascontiguousarray(x, dtype=np.uint32)


def store_error(t, y):
    return np.abs(y) * 2.0 ** (-24 if t == 0 else -11) + (0 if t == 0 else 2.0 ** -25)


def close(got, want, tol):
    err = np.abs(got - want)
    ok = err <= tol
    assert ok.all(), (float(np.nanmax(err)), float(np.nanmax(err - tol)), int((~ok).sum()))


class Cache:
    """Random caches of n pages, on both sides."""

    def __init__(self, ctx, rng, n, nkv, hd, fmt, odd_scales=False, spread=1):
        self.ctx, self.n, self.nkv, self.hd, self.fmt = ctx, n, nkv, hd, fmt
        if fmt == I8:
            self.k, self.v = (rng.integers(-127, 128, (nkv, n * 16, hd)).astype(np.int8).view(np.uint8) for _ in range(2))
        else:
            self.k, self.v = (ref.encode(np.clip(rng.normal(size=(nkv, n * 16, hd)) * 100, -448, 448), fmt) for _ in range(2))
        base = -6 if fmt == I8 else -7
        self.ks, self.vs = ((2.0 ** (base + rng.integers(-spread, spread + 1, (n, nkv)))).astype(np.float32) for _ in range(2))
        if odd_scales:
            self.ks, self.vs = ((s * rng.uniform(1, 2, s.shape)).astype(np.float32) for s in (self.ks, self.vs))
        self.put()

    def put(self):
        self.b = [self.ctx.upload(x) for x in (self.k, self.v, self.ks, self.vs)]

    def batch(self, zh, tables, lens, starts=None):
        c = self.ctx
        return zh.Kv8Batch(*self.b, c.upload(u32(tables)), c.upload(u32(lens)),
                           row_start=None if starts is None else c.upload(u32(starts)), n_seq=len(lens),
                           table_stride=tables.shape[1], cache_tokens=16 * self.n, n_kv_heads=self.nkv,
                           head_dim=self.hd, type=self.fmt)

    def get(self):
        return (self.b[0].download(np.uint8, self.k.size).reshape(self.k.shape),
                self.b[1].download(np.uint8, self.v.size).reshape(self.v.shape),
                self.b[2].download(np.float32, self.ks.size).reshape(self.ks.shape),
                self.b[3].download(np.float32, self.vs.size).reshape(self.vs.shape))


def tables_for(rng, lens, extra=0):
    """Page tables of sequences of the given lengths over shuffled pages: (tables, pages of the cache)."""
    pages = [-(-int(n) // 16) for n in lens]
    total = max(sum(pages), 1) + extra
    perm, at = rng.permutation(total), 0
    t = np.full((len(lens), max(max(pages), 1)), 0, dtype=np.uint32)
    for s, n in enumerate(pages):
        t[s, :n] = perm[at:at + n]
        at += n
    return t, total


# ---------------------------------------------------------------------------
# q/k norm + rotation + quantised write
# ---------------------------------------------------------------------------
WRITE = [  # counts, lens, q heads, kv heads, head_dim, rope_dim, type, q type, norm
    ([1], [1], 4, 2, 128, 128, 0, 0, True),
    ([1], [17], 4, 2, 64, 64, 0, 0, True),
    ([1, 1, 1], [40, 16, 33], 32, 8, 128, 128, 0, 1, True),
    ([1] * 70, None, 5, 1, 128, 64, 1, 1, True),
    ([16, 5, 40], [16, 25, 47], 8, 4, 128, 128, 0, 0, True),
    ([100, 0, 3, 31, 1], [131, 9, 4, 31, 1], 7, 7, 64, 32, 1, 0, False),
    ([1, 200, 2, 77], [300, 205, 18, 77], 20, 2, 128, 24, 1, 1, True),
    ([33] * 130, None, 2, 1, 64, 64, 0, 1, True),
    ([19, 13], [90000, 131072], 3, 3, 128, 128, 0, 0, True),
    ([9], [9], 4, 2, 128, 0, 0, 1, True),
    ([12, 12], [50, 12], 17, 1, 64, 16, 1, 1, False),
]


def ragged(rng, counts, lens):
    return np.array([c + int(rng.integers(0, 60)) for c in counts] if lens is None else lens)


@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("case", WRITE)
def test_write(zh, ctx, fmt, case):
    counts, lens, nq, nkv, hd, rd, t, qt, norm = case
    rng = np.random.default_rng(len(counts) * 7 + nq)
    lens = ragged(rng, counts, lens)
    # (tables name pages where the call writes; the others' entries are 0)
    S, T = len(counts), sum(counts)
    tables = np.zeros((S, -(-int(lens.max()) // 16)), dtype=np.uint32)
    used = [range((n - c) // 16, -(-n // 16)) if c else range(0) for n, c in zip(lens, counts)]
    total = sum(len(r) for r in used) + 3
    perm, at = rng.permutation(total), 0
    for s, r in enumerate(used):
        tables[s, r.start:r.stop] = perm[at:at + len(r)]
        at += len(r)
    cache = Cache(ctx, rng, total, nkv, hd, fmt)
    decode = all(c == 1 for c in counts)
    starts = None if decode else np.concatenate([[0], np.cumsum(counts)])
    kv = cache.batch(zh, tables, lens, starts)
    width = (nq + 2 * nkv) * hd
    x = (rng.normal(size=(T, width)) * rng.choice([0.3, 2, 9], (T, 1))).astype(NP_TYPE[t])
    wq, wk = ((1 + 0.2 * rng.normal(size=hd)).astype(np.float32) for _ in range(2))
    freq = (1e6 ** (-np.arange(0, max(rd, 2), 2) / max(rd, 2))).astype(np.float32)
    xb, size = ctx.upload(x), x.itemsize
    out = ctx.upload(np.full((T, nq * hd), 77, dtype=NP_TYPE[qt]))
    rows = zh.QkvRows(q=xb, k=xb, v=xb, k_off=nq * hd * size, v_off=(nq + nkv) * hd * size, q_stride=width,
                      k_stride=width, v_stride=width, type=t, q_out=out, q_out_type=qt, pos=None, n_rows=T,
                      n_q_heads=nq, rope_dim=rd, inv_freq=ctx.upload(freq) if rd else None,
                      q_norm_w=ctx.upload(wq) if norm else None, k_norm_w=ctx.upload(wk) if norm else None, eps=1e-6)
    ctx.qk_norm_rope_kv8_write_batched(kv, rows)
    ctx.sync()
    pos = np.concatenate([np.arange(n - c, n) for n, c in zip(lens, counts)])
    seq = np.repeat(np.arange(S), counts)
    h = x.reshape(T, nq + 2 * nkv, hd)
    q = ref.turned(h[:, :nq], wq if norm else None, freq, pos, 1e-6, rd)
    plain = ref.turned(h[:, :nq], wq if norm else None, freq, pos, 1e-6, 0)
    mag = np.abs(plain)
    if rd:
        mag[..., :rd // 2] = mag[..., rd // 2:rd] = mag[..., :rd // 2] + mag[..., rd // 2:rd]
    close(out.download(NP_TYPE[qt], T * nq * hd).reshape(q.shape).astype(np.float64), q,
          2.0 ** -19 * mag + store_error(qt, q))
    k = ref.turned(h[:, nq:nq + nkv], wk if norm else None, freq, pos, 1e-6, rd)
    got = cache.get()
    for codes, scales, new, gc, gs in ((cache.k, cache.ks, k, got[0], got[2]),
                                       (cache.v, cache.vs, h[:, nq + nkv:].astype(np.float64), got[1], got[3])):
        codes, scales = codes.copy(), scales.copy()
        for page in sorted({(s, p // 16) for s, p in zip(seq, pos)}):
            phys = tables[page]
            which = np.flatnonzero((seq == page[0]) & (pos // 16 == page[1]))
            for hh in range(nkv):
                block = slice(phys * 16, phys * 16 + 16)
                codes[hh, block], scales[phys, hh] = ref.store_page(codes[hh, block], scales[phys, hh], fmt,
                                                                    list(pos[which] % 16), new[which, hh])
        assert np.array_equal(gs, scales)
        assert np.array_equal(ref.decode(gc, fmt), ref.decode(codes, fmt))


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
ATTN = [  # counts, lens, heads per kv head, kv heads, head_dim
    ([1], [1], 1, 1, 128),
    ([1], [16], 4, 2, 64),
    ([1, 1, 1], [200, 0, 33], 4, 8, 128),
    ([1] * 5, [1000, 17, 700, 64, 65], 5, 2, 128),
    ([1] * 3, [5000, 300, 1], 16, 1, 64),
    ([1], [9000], 32, 1, 128),
    ([1] * 40, None, 3, 4, 64),
    ([3, 1, 5], [130, 64, 5], 4, 2, 128),
    ([2], [2], 1, 1, 64),
    ([7, 7], [1023, 800], 4, 2, 64),
    ([33, 0, 2], [33, 12, 700], 4, 2, 128),
    ([50], [2000], 7, 1, 128),
    ([300, 1, 65], [300, 900, 400], 4, 2, 64),
    ([129], [640], 1, 3, 128),
    ([20], [50], 71, 1, 64),
    ([600], [2500], 2, 2, 128),
]


def attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts, scale=0.0, q=None, max_rows=None, max_len=None,
           check=True, **more):
    T, nh = int(sum(counts)), G * cache.nkv
    q = (rng.normal(size=(T, nh, cache.hd)) * 2).astype(NP_TYPE[t]) if q is None else q
    kv = cache.batch(zh, tables, lens, starts)
    most, longest = max_rows or max(counts), max_len or max(1, int(max(lens)))
    ws = ctx.alloc(ctx.flash_attn_kv8_ws(kv, nh, T, most, longest))
    out = ctx.upload(np.full((T, nh * cache.hd), 77, dtype=NP_TYPE[t]))
    rows = zh.AttnRows(q=ctx.upload(q), out=out, ws=ws, n_rows=T, max_rows=most, max_len=longest, n_heads=nh, type=t,
                       attn_scale=scale, **more)
    ctx.flash_attn_kv8(kv, rows)
    if check:
        ctx.sync()
    return q, out.download(NP_TYPE[t], T * nh * cache.hd).reshape(q.shape).astype(np.float64)


def expect(cache, tables, q, counts, lens, scale):
    first, parts = 0, []
    for s, (c, n) in enumerate(zip(counts, lens)):
        parts.append(ref.attention(q[first:first + c], cache.k, cache.v, cache.ks, cache.vs, tables[s], c, int(n), scale,
                                   cache.fmt))
        first += c
    return [np.concatenate([p[i] for p in parts]) for i in range(4)]


def tolerance(cache, t, want, mag, unit, big, lens, odd=False, floor=-39):
    e = np.abs(np.log2(cache.vs)).max()
    tol = mag * (2.0 ** -17 * 1.45 * big[..., None] + (max(lens) / 32 + 84 + 2 * e) * 2.0 ** -23 + (2.0 ** -19 if odd else 0)) + 2.0 ** floor * unit
    return tol + (2.0 ** -11 * mag + store_error(1, want) if t else 0)


@pytest.mark.parametrize("t", [0, 1])
@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("case", ATTN)
def test_attention(zh, ctx, fmt, t, case):
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + G)
    lens = ragged(rng, counts, lens)
    tables, total = tables_for(rng, lens, 2)
    cache = Cache(ctx, rng, total, nkv, hd, fmt)
    starts = None if all(c == 1 for c in counts) else np.concatenate([[0], np.cumsum(counts)])
    q, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, t, starts)
    want, *terms = expect(cache, tables, q, counts, lens, hd ** -0.5)
    tiled = max(counts) * G > 128
    close(got, want, tolerance(cache, t, want, *terms, lens, floor=-29 if tiled else -39))

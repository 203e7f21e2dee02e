"""The batched operators over a paged KV cache on the GPU, against plain numpy
in 64 bits on the same fp16 cache and page tables.

Tolerances. An f32 rounding is off by 2^-24 of the value, an fp16 one by 2^-11
(or 2^-25 below the normal range).
  rope: mean of squares, square root, division and the products before the
    rotation: at most 24 roundings of 2^-24; the angle enters as a fraction of a
    turn within 2^-26 (2^-23.3 radians), its sine and cosine within 2^-22; three
    roundings of the rotation. Together less than 2^-19 (|a| + |b|) for the pair
    (a, b), and the store's own rounding.
  attention: a score is off by at most 2^-18 A, A = 1.45 scale sum |q_i k_i| of
    its row's largest (q in two pieces: 2^-22; 8 chained matrix instructions of
    32 products, each step within 2^-22 of the sum of magnitudes; the scaling and
    the subtraction of the maximum 2^-23 each), and with it a weight by 2^-18 A
    relative plus 2^-21 (exp2, two pieces). That enters the numerator and the sum
    of weights; the sums over n tokens add n / 32 + 64 steps of 2^-23:
    |error| <= W (2^-17 A + (n / 32 + 80) 2^-23), W = sum w |v| of the output.
    ZH_F16 adds 2^-11 W for the weights in one piece and the store's rounding.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF


@pytest.fixture(scope="module")
def zh():
    import zinc_amd
    return zinc_amd


@pytest.fixture()
def ctx(zh):
    c = zh.Context(0)
    yield c
    c.close()


NP_TYPE = {0: np.float32, 1: np.float16}


def store_error(t, y):
    """The rounding of a stored y of type t."""
    return np.abs(y) * 2.0 ** (-24 if t == 0 else -11) + (0 if t == 0 else 2.0 ** -25)


def close(got, want, tol, where=...):
    err = np.abs(got - want)
    ok = (err <= tol)[where].all()
    assert ok, (float(np.nanmax(err)), float(np.nanmax((err - tol)[where])), int((~(err <= tol))[where].sum()))


# ---------------------------------------------------------------------------
# page copies
# ---------------------------------------------------------------------------
def copied(caches, dst, src, nkv, hd):
    out = []
    for c in caches:
        c = c.copy().reshape(nkv, -1, 16, hd)
        c[:, dst] = c[:, src]
        out.append(c.reshape(-1))
    return out


@pytest.mark.parametrize("n_caches,nkv,hd,pool,n", [
    (1, 1, 64, 4, 1), (2, 8, 128, 40, 13), (97, 2, 64, 9, 3), (3, 3, 80, 700, 300), (2, 1, 2, 30, 11), (4, 5, 6, 20, 9),
    (2, 2, 512, 12, 5), (2, 4, 128, 1100, 513), (4, 1, 2, 4000, 1990),
    (64, 1, 2, 3100, 1445), (65, 1, 2, 1500, 700), (3, 1, 2, 65536 + 40, 270), (1, 1, 64, 65536, 30)])
def test_copy_pages(zh, ctx, n_caches, nkv, hd, pool, n):
    rng = np.random.default_rng(pool + n)
    caches = [rng.integers(0, 1 << 16, nkv * pool * 16 * hd).astype(np.uint16) for _ in range(n_caches)]
    bufs = [ctx.upload(c) for c in caches]
    s = zh.KvCaches(bufs, pool * 16, nkv, hd)
    perm = rng.permutation(pool)
    dst, src = perm[:n], rng.choice(perm[n:], n)  # a source may go to several places
    ctx.kv_copy_pages(s, s, dst, src)
    for b, want in zip(bufs, copied(caches, dst, src, nkv, hd)):
        assert np.array_equal(b.download(np.uint16, want.size), want)


def test_copy_between_caches_of_other_sizes(zh, ctx):
    rng = np.random.default_rng(3)
    nkv, hd = 2, 64
    a = [rng.integers(0, 1 << 16, (nkv, 10, 16, hd)).astype(np.uint16) for _ in range(2)]
    b = [rng.integers(0, 1 << 16, (nkv, 7, 16, hd)).astype(np.uint16) for _ in range(2)]
    A, B = [ctx.upload(x) for x in a], [ctx.upload(x) for x in b]
    ctx.kv_copy_pages(zh.KvCaches(B, 7 * 16, nkv, hd),
                      zh.KvCaches(A, 160, nkv, hd), [6, 0, 3], [9, 3, 0])
    for x, y, Y in zip(a, b, B):
        y[:, [6, 0, 3]] = x[:, [9, 3, 0]]
        assert np.array_equal(Y.download(np.uint16, y.size), y.reshape(-1))
    for x, X in zip(a, A):
        assert np.array_equal(X.download(np.uint16, x.size), x.reshape(-1))


def test_copy_refusal_changes_nothing_and_none_is_fine(zh, ctx):
    c = np.arange(4 * 16 * 64, dtype=np.uint16)
    b = ctx.upload(c)
    s = zh.KvCaches([b], 64, 1, 64)
    for d, q in (([1, 1], [2, 3]), ([1, 2], [2, 3]), ([1], [4])):
        with pytest.raises(zh.ZincError) as e:
            ctx.kv_copy_pages(s, s, d, q)
        assert e.value.name == "InvalidArgument"
    ctx.kv_copy_pages(s, s, [], [])
    ctx.sync()
    assert np.array_equal(b.download(np.uint16, c.size), c)


# ---------------------------------------------------------------------------
# q/k norm + rotation + KV write
# ---------------------------------------------------------------------------
def rope64(x, w, freq, pos, eps, rd):
    """x [T][heads][hd]: the rotated rows and sum |a| + |b| of each pair."""
    x = x.astype(np.float64)
    if w is not None:
        x = w.astype(np.float64) * (x / np.sqrt((x * x).mean(-1, keepdims=True) + eps))
    y, mag = x.copy(), np.abs(x)
    h = rd // 2
    if h:
        th = (pos.astype(np.float64)[:, None] * freq.astype(np.float64))[:, None]
        a, b = x[..., :h], x[..., h:rd]
        y[..., :h], y[..., h:rd] = a * np.cos(th) - b * np.sin(th), a * np.sin(th) + b * np.cos(th)
        mag[..., :h] = mag[..., h:rd] = np.abs(a) + np.abs(b)
    return y, mag


ROPE = [  # rows, seqs, q heads, kv heads, head_dim, rope_dim, type, q type, norm, stacked
    (1, 1, 4, 2, 128, 128, 0, 0, True, False),
    (5, 3, 32, 8, 128, 128, 0, 0, True, True),
    (33, 4, 10, 2, 128, 64, 0, 1, True, True),
    (70, 2, 7, 7, 64, 64, 1, 1, True, True),
    (300, 9, 8, 1, 64, 32, 1, 0, False, True),
    (19, 19, 6, 3, 256, 256, 0, 1, True, True),
    (9, 2, 3, 1, 80, 80, 0, 0, True, False),     # no power of two
    (9, 2, 3, 1, 96, 40, 1, 1, True, True),
    (12, 3, 2, 2, 6, 4, 1, 1, True, True),       # odd sizes, 2-byte aligned rows
    (4, 1, 2, 1, 2, 2, 0, 0, False, False),
    (8, 2, 4, 4, 512, 512, 0, 0, True, True),
    (8, 2, 4, 2, 128, 0, 0, 1, True, True),      # norm alone
    (40, 5, 16, 4, 128, 128, 1, 1, False, True),
    (1030, 3, 5, 5, 128, 128, 0, 1, True, True),
]


@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c)))
def test_rope_batched(zh, ctx, case):
    T, S, nq, nkv, hd, rd, ti, tq, norm, stacked = case
    rng = np.random.default_rng(T * 7 + hd)
    far = 200000
    stride = far // 16 + 1
    # rows of sequences in any order, distinct positions, some rows padded
    seq = rng.integers(0, S, T)
    pos = rng.choice(far, T, replace=False)
    pos[0] = far - 1
    pages_needed = sorted({(s, p // 16) for s, p in zip(seq, pos)})
    pool = len(pages_needed) + 2
    perm = rng.permutation(pool).astype(np.uint32)
    tables = np.full((S, stride), pool + 7, dtype=np.uint32)  # (entries that no row uses lie outside)
    for i, (s, p) in enumerate(pages_needed):
        tables[s, p] = perm[i]
    pad = rng.random(T) < 0.1
    pad[0] = False
    tokens = pool * 16
    kc, vc = (rng.standard_normal((nkv, tokens, hd)).astype(np.float16) for _ in range(2))
    qkv = (rng.standard_normal((T, nq + 2 * nkv, hd)) * 3).astype(NP_TYPE[ti])
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    freq = (1e6 ** (-np.arange(0, rd, 2) / max(rd, 1))).astype(np.float32)
    size, width = np.dtype(NP_TYPE[ti]).itemsize, (nq + 2 * nkv) * hd
    gap = 8 if stacked else 0
    out0 = rng.standard_normal((T + 1, nq * hd + gap)).astype(NP_TYPE[tq])
    u = ctx.upload
    kcb, vcb = u(kc), u(vc)
    kv = zh.KvBatch(kcb, vcb, u(tables), S, stride, tokens, nkv, hd)
    if stacked:
        X = u(qkv)
        where = dict(q=X, k=X, v=X, k_off=nq * hd * size, v_off=(nq + nkv) * hd * size, q_stride=width, k_stride=width,
                     v_stride=width)
    else:
        where = dict(q=u(qkv[:, :nq]), k=u(qkv[:, nq:nq + nkv]), v=u(qkv[:, nq + nkv:]))
    outb = u(out0)
    rows = zh.QkvRows(q_out=outb, q_out_stride=nq * hd + gap, pos=u(np.where(pad, NONE, pos).astype(np.uint32)),
                      seq=u(seq.astype(np.uint32)), n_rows=T, n_q_heads=nq, rope_dim=rd,
                      inv_freq=u(freq) if rd else None, q_norm_w=u(qw) if norm else None,
                      k_norm_w=u(kw) if norm else None, type=ti, q_out_type=tq, eps=1e-5, **where)
    ctx.qk_norm_rope_kv_write_batched(kv, rows)
    ctx.sync()
    got = outb.download(NP_TYPE[tq], out0.size).reshape(out0.shape)
    want, mag = rope64(qkv[:, :nq], qw if norm else None, freq, pos, 1e-5, rd)
    live = ~pad
    err = np.abs(got[:T, :nq * hd].reshape(T, nq, hd).astype(np.float64) - want)
    assert (err <= mag * 2.0 ** -19 + store_error(tq, want))[live].all(), err[live].max()
    # padded rows, the gaps and the row behind are as they were
    assert np.array_equal(got[:T][pad], out0[:T][pad]) and np.array_equal(got[T], out0[T])
    assert np.array_equal(got[:, nq * hd:], out0[:, nq * hd:])
    k64, kmag = rope64(qkv[:, nq:nq + nkv], kw if norm else None, freq, pos, 1e-5, rd)
    wk, wv, tol = kc.astype(np.float64), vc.astype(np.float64), np.zeros(kc.shape)
    for t in np.flatnonzero(live):
        slot = int(tables[seq[t], pos[t] // 16]) * 16 + pos[t] % 16
        wk[:, slot], wv[:, slot] = k64[t], qkv[t, nq + nkv:].astype(np.float16)
        tol[:, slot] = kmag[t] * 2.0 ** -19 + store_error(1, k64[t])
    gk, gv = (b.download(np.float16, kc.size).reshape(kc.shape).astype(np.float64) for b in (kcb, vcb))
    assert (np.abs(gk - wk) <= tol).all() and np.array_equal(gv, wv)


def test_rope_in_place_and_like_the_single_token_entry(zh, ctx):
    """One row through both entries (near positions, where a 32-bit angle is
    good to 2^-24 of itself: at most 40 radians), q in place."""
    rng = np.random.default_rng(1)
    nq, nkv, hd, tokens = 8, 2, 128, 64
    q, k, v = (rng.standard_normal(n * hd).astype(np.float32) for n in (nq, nkv, nkv))
    qw, kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    freq = (1e6 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    pages = np.array([2, 0, 3, 1], dtype=np.uint32)
    u = ctx.upload
    got = []
    for batched in (False, True):
        Q, kc, vc = u(q), u(np.zeros((nkv, tokens, hd), np.float16)), u(np.zeros((nkv, tokens, hd), np.float16))
        if batched:
            kv = zh.KvBatch(kc, vc, u(pages), 1, 4, tokens, nkv, hd)
            ctx.qk_norm_rope_kv_write_batched(kv, zh.QkvRows(
                q=Q, k=u(k), v=u(v), q_out=Q, pos=u(np.array([39], np.uint32)), n_rows=1, n_q_heads=nq, rope_dim=hd,
                inv_freq=u(freq), q_norm_w=u(qw), k_norm_w=u(kw), eps=1e-6))
        else:
            ctx.qk_norm_rope_kv_write(Q, u(qw), u(k), u(kw), u(v), u(freq), kc, vc, u(pages), 4, tokens, nq, nkv, hd,
                                      39, 1e-6)
        got.append((Q.download(np.float32, q.size), kc.download(np.float16, nkv * tokens * hd),
                    vc.download(np.float16, nkv * tokens * hd)))
    mag = 2 * np.abs(q).max() * 1.5 * 2
    assert np.abs(got[0][0] - got[1][0]).max() <= mag * (39 * 2.0 ** -24 + 2.0 ** -18)
    assert np.abs(got[0][1].astype(np.float64) - got[1][1]).max() <= mag * (39 * 2.0 ** -24 + 2.0 ** -18 + 2.0 ** -10)
    assert np.array_equal(got[0][2], got[1][2])


def test_rope_rows_outside_are_left_out_and_reported(zh, ctx):
    rng = np.random.default_rng(2)
    nq, nkv, hd, tokens, S, stride = 2, 1, 64, 64, 2, 3
    x = rng.standard_normal((5, 4, hd)).astype(np.float32)
    u = ctx.upload
    kc0 = rng.standard_normal((nkv, tokens, hd)).astype(np.float16)
    kc, vc = u(kc0), u(kc0)
    tables = np.array([[0, 1, 4], [2, 0xFFFFFFFF, 0x10000000]], dtype=np.uint32)  # 4 and the last two lie outside
    seq = np.array([0, 0, 1, 1, 2], dtype=np.uint32)
    pos = np.array([48, 33, 17, 40, 3], dtype=np.uint32)  # past the table, page 4, no page, wrapped page, no sequence
    out = ctx.alloc(4 * 5 * nq * hd)
    X = u(x)
    kv = zh.KvBatch(kc, vc, u(tables), S, stride, tokens, nkv, hd)
    rows = dict(q=X, k=X, v=X, k_off=4 * 2 * hd, v_off=4 * 3 * hd, q_stride=4 * hd, k_stride=4 * hd, v_stride=4 * hd,
                q_out=out, seq=u(seq), pos=u(pos), n_q_heads=nq)
    ctx.qk_norm_rope_kv_write_batched(kv, zh.QkvRows(n_rows=5, **rows))
    with pytest.raises(zh.ZincError) as e:
        ctx.sync()
    assert e.value.name == "InvalidArgument"
    ctx.sync()  # reported once
    assert np.array_equal(out.download(np.float32, 5 * nq * hd).reshape(5, nq, hd), x[:, :nq])
    for b in (kc, vc):
        assert np.array_equal(b.download(np.float16, kc0.size).reshape(kc0.shape), kc0)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def attend64(q, kc, vc, tables, lens, scale, t, P=0, only=None):
    """(out, bound) of the module's formula; q [S][nh][hd]. The first P tokens
    of the sequences that long are read through sequence 0's table. only: the
    sequences worked out."""
    S, nh, hd = q.shape
    nkv = kc.shape[0]
    G = nh // nkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for s in range(S) if only is None else only:
        n = int(lens[s])
        if n == 0:
            continue
        tk = np.arange(n)
        via = np.where((tk < P) & (n >= P), 0, s)
        at = tables[via, tk // 16].astype(np.int64) * 16 + tk % 16
        for g in range(nkv):
            hs = slice(g * G, g * G + G)
            k, v = kc[g, at].astype(np.float64), vc[g, at].astype(np.float64)
            x = q[s, hs].astype(np.float64)
            sc = x @ k.T * scale
            A = 1.45 * abs(scale) * (np.abs(x) @ np.abs(k).T).max(1, keepdims=True)
            w = np.exp(sc - sc.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            out[s, hs], W = w @ v, w @ np.abs(v)
            tol[s, hs] = W * (2.0 ** -17 * A + (n / 32 + 80) * 2.0 ** -23) + store_error(t, out[s, hs])
            if t == 1:
                tol[s, hs] += W * 2.0 ** -11
    return out, tol


def make(rng, S, nkv, hd, P, lens, shared=True, spare=2, poison=True):
    """Caches and tables of sequences sharing their first P tokens; every slot
    that no sequence uses, and the tables' unused entries, hold what must not
    enter a result."""
    lens = np.asarray(lens)
    M = max(int(lens.max()), P, 1)
    stride = -(-M // 16)
    full = P // 16 if shared else 0
    own = [max(0, -(-int(n) // 16) - full) if n >= P else -(-int(n) // 16) for n in lens]
    own[0] = max(own[0], stride - full) if P else own[0]  # sequence 0's table covers the prefix
    total = full + sum(own) + spare
    perm = rng.permutation(total).astype(np.uint32)
    tables = np.full((S, stride), 0xFFFFFFF0, dtype=np.uint32)
    kc = np.full((nkv, total * 16, hd), np.nan if poison else 1.0, dtype=np.float16)
    vc = kc.copy()
    if poison:
        vc[:, ::3] = np.inf
    at = full
    for s in range(S):
        k = full if lens[s] >= P or s == 0 else 0
        tables[s, :k] = perm[:k]
        tables[s, k:k + own[s]] = perm[at:at + own[s]]
        at += own[s]
    base = [rng.standard_normal((P, nkv, hd), dtype=np.float32).astype(np.float16) for _ in range(2)]
    for s in range(S):
        n = max(int(lens[s]), P) if s == 0 else int(lens[s])
        first = full * 16 if s and n >= P else 0  # (the shared pages are written once)
        t = np.arange(first, n)
        slots = tables[s, t // 16].astype(np.int64) * 16 + t % 16
        for c, b in zip((kc, vc), base):
            x = rng.standard_normal((n - first, nkv, hd), dtype=np.float32).astype(np.float16)
            if n >= P:
                x[:P - first] = b[first:]
            c[:, slots] = x.transpose(1, 0, 2)
    return kc, vc, tables, total * 16, M


def run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, scale=0.0, gap=0, in_place=False, expect_error=False):
    S, nh, hd = q.shape
    u = ctx.upload
    kv = zh.KvBatch(u(kc), u(vc), u(tables), S, tables.shape[1], kc.shape[1], kc.shape[0], hd)
    rng = np.random.default_rng(9)
    buf = rng.standard_normal((S + 1, nh * hd + gap)).astype(NP_TYPE[t])
    buf[:S, :nh * hd] = q.reshape(S, -1)
    out0 = buf.copy() if in_place else rng.standard_normal(buf.shape).astype(NP_TYPE[t])
    Q = u(buf)
    O = Q if in_place else u(out0)
    n = ctx.flash_decode_shared_ws(kv, nh, P, M)
    assert n > 0
    guard = np.full(n // 4 + 64, 0x5A5A5A5A, dtype=np.uint32)
    ws = u(guard)
    rows = zh.DecodeRows(q=Q, out=O, seq_lens=u(np.asarray(lens, dtype=np.uint32)), ws=ws, n_heads=nh, prefix_len=P,
                         max_len=M, type=t, q_stride=nh * hd + gap, out_stride=nh * hd + gap, attn_scale=scale)
    ctx.flash_decode_shared(kv, rows)
    if expect_error:
        with pytest.raises(zh.ZincError) as e:
            ctx.sync()
        assert e.value.name == "InvalidArgument"
    ctx.sync()
    got = O.download(NP_TYPE[t], out0.size).reshape(out0.shape)
    assert np.array_equal(got[:, nh * hd:], out0[:, nh * hd:]) and np.array_equal(got[S], out0[S])
    assert (ws.download(np.uint32, guard.size)[(n + 3) // 4:] == 0x5A5A5A5A).all()
    if not in_place:
        ctx.flash_decode_shared(kv, rows)  # the same bits again
        if expect_error:
            with pytest.raises(zh.ZincError):
                ctx.sync()
        assert np.array_equal(O.download(NP_TYPE[t], out0.size).view(np.uint8), got.reshape(-1).view(np.uint8))
    return got[:S, :nh * hd].reshape(S, nh, hd).astype(np.float64)


ATTN = [  # q heads, kv heads, head_dim, prefix, lengths
    (4, 4, 128, 0, [1]),
    (32, 8, 128, 0, [17]),
    (32, 8, 128, 16, [17, 16]),
    (10, 2, 128, 200, [201, 240, 215]),
    (3, 1, 64, 33, [33, 34, 49, 65, 33]),
    (16, 1, 64, 0, [0, 5, 100, 0, 31, 32, 33]),
    (16, 1, 128, 500, [700, 501, 500, 631]),
    (8, 8, 128, 130, [300, 131, 20, 0, 129, 130, 131]),          # some shorter than the prefix
    (7, 7, 64, 1000, [1000, 3, 1000, 999]),
    (32, 4, 128, 1500, [1500 + 37 * i % 200 for i in range(21)]),  # 168 rows a kv head
    (16, 8, 64, 777, [778 + 5 * i for i in range(70)]),
    (14, 2, 128, 0, [4097, 63, 1024]),
    (12, 4, 128, 2049, [2049 + 1 + i % 3 for i in range(40)]),
    (8, 1, 128, 640, [640] * 64),                                 # nothing of their own
    (2, 2, 128, 9000, [9001, 9100]),
    (48, 4, 128, 300, [301 + i for i in range(90)]),              # 1080 rows a kv head
]


@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
def test_attention(zh, ctx, case, t):
    nh, nkv, hd, P, lens = case
    rng = np.random.default_rng(nh * 100 + P)
    kc, vc, tables, _, M = make(rng, len(lens), nkv, hd, P, lens)
    q = (rng.standard_normal((len(lens), nh, hd)) * 1.5).astype(NP_TYPE[t])
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, gap=8 * (P % 2))
    want, tol = attend64(q, kc, vc, tables, lens, hd ** -0.5, t, P)
    close(got, want, tol)


TILED = [  # many rows over a long prefix: K and V through LDS, 128 or 256 rows a workgroup
    (64, 4, 128, 1237, [0, 1237, 5] + [1238 + 3 * i for i in range(60)]),   # 1008 rows, 4 workgroups
    (64, 4, 128, 1907, [1907, 3] + [1908 + i % 90 for i in range(60)]),     # 992 rows, f32 too
    (128, 8, 128, 4701, [4701 + 17 * i for i in range(8)]),                 # 128 rows
    (48, 8, 64, 12601, [12650, 12601, 400, 12640, 12602, 12700, 13000]),    # 42 rows
    (16, 4, 64, 5000, [5001 + i for i in range(70)]),                       # 280 rows
    (64, 64, 64, 4510, [4511 + i % 5 for i in range(130)]),                 # parts of more than 64 pages
    (33, 33, 128, 7000, [7001 + 70 * i % 600 for i in range(34)]),          # own tokens in parts of their own
    # long enough for tiles in f32 too
    (128, 8, 128, 12001, [12001 + 17 * i for i in range(8)]),
    (64, 4, 128, 3137, [3137, 3] + [3138 + i % 90 for i in range(60)]),
    (48, 8, 64, 24001, [24050, 24001, 400, 24040, 24002, 24100, 24400]),
    (33, 33, 128, 7741, [7742 + 90 * i % 1300 for i in range(34)]),
]


@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("case", TILED, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
def test_attention_of_many_rows(zh, ctx, case, t):
    nh, nkv, hd, P, lens = case
    rng = np.random.default_rng(nh * 100 + P)
    kc, vc, tables, _, M = make(rng, len(lens), nkv, hd, P, lens)
    q = (rng.standard_normal((len(lens), nh, hd)) * 1.5).astype(NP_TYPE[t])
    scale = -0.11 if nh == 16 else hd ** -0.5
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, scale=scale)
    assert np.isfinite(got).all()
    only = sorted({0, 1, 2, len(lens) // 2, len(lens) - 1})
    want, tol = attend64(q, kc, vc, tables, lens, scale, t, P, only)
    close(got[only], want[only], tol[only])


@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
def test_attention_in_tiles_of_odd_queries_and_a_bad_page(zh, ctx, t):
    """992 rows over a prefix of 3137 tokens: a query of f16's smallest values, one
    with a NaN (no other row's), and a page of the prefix outside the cache."""
    rng = np.random.default_rng(22)
    P, lens = 3137, [3138 + i % 40 for i in range(62)]
    kc, vc, tables, _, M = make(rng, 62, 4, 128, P, lens, poison=False)
    q = rng.standard_normal((62, 64, 128)).astype(NP_TYPE[t])
    q[5] *= NP_TYPE[t](2.0 ** -20)
    x = q.copy()
    x[7, 9, 3] = np.nan
    tables[0, 100] = 0xFFFFFFFF
    got = run_attention(zh, ctx, x, kc, vc, tables, lens, P, M, t, expect_error=True)
    tables[0, 100] = 0
    only = [0, 5, 7, 61]
    want, tol = attend64(q, kc, vc, tables, lens, 128 ** -0.5, t, P, only)
    ok = np.ones(got.shape, bool)
    ok[7, 9] = False
    assert np.isnan(got[7, 9]).all()
    close(got[only], want[only], tol[only], ok[only])


@pytest.mark.parametrize("P", [1408, 2944])  # (f16 in tiles, f32 too)
def test_attention_rescales_when_later_scores_are_larger(zh, ctx, P):
    """Scores that grow along a prefix by about 2^15 in all, in tiles and
    streamed: the running maximum moves again and again."""
    rng = np.random.default_rng(21)
    lens = [P + 2 + i for i in range(64)]
    kc, vc, tables, _, M = make(rng, 64, 4, 128, P, lens)
    q = rng.standard_normal((64, 64, 128)).astype(np.float16)
    t = np.arange(P)
    slots = tables[0, t // 16].astype(np.int64) * 16 + t % 16
    u = rng.standard_normal(128)
    u /= np.linalg.norm(u)
    q = (q + 6 * u).astype(np.float16)  # every row along u, every K further along it
    kc[:, slots] = (kc[:, slots].astype(np.float64) + (t / P * 20)[None, :, None] * u).astype(np.float16)
    for typ in (0, 1):
        x = q.astype(NP_TYPE[typ])
        for n in (64, 3):  # 1024 rows a kv head, and 48
            got = run_attention(zh, ctx, x[:n], kc, vc, tables[:n], lens[:n], P, M, typ)
            only = [0, n - 1]
            want, tol = attend64(x[:n], kc, vc, tables[:n], lens[:n], 128 ** -0.5, typ, P, only)
            close(got[only], want[only], tol[only])


@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
def test_attention_in_place_other_scale_and_room_behind(zh, ctx, t):
    rng = np.random.default_rng(4)
    lens = [90, 61, 77]
    kc, vc, tables, _, M = make(rng, 3, 2, 64, 48, lens)
    q = rng.standard_normal((3, 6, 64)).astype(NP_TYPE[t])
    wide = np.full((3, 40), 0xFFFFFFFF, dtype=np.uint32)  # a table and a max_len with room for more tokens
    wide[:, :tables.shape[1]] = tables
    for in_place in (False, True):
        got = run_attention(zh, ctx, q, kc, vc, wide, lens, 48, 640, t, scale=0.31, gap=16, in_place=in_place)
        want, tol = attend64(q, kc, vc, tables, lens, 0.31, t)
        close(got, want, tol)


@pytest.mark.parametrize("size", [1e-30, 3e-6, 1.0, 4e5, 1e30])
def test_attention_of_f32_queries_of_any_size(zh, ctx, size):
    """q far outside fp16's range (the scale takes it back)."""
    rng = np.random.default_rng(6)
    lens = [140, 139]
    kc, vc, tables, _, M = make(rng, 2, 1, 128, 100, lens)
    q = (rng.standard_normal((2, 4, 128)) * size).astype(np.float32)
    scale = float(np.float32(0.09 / size))
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, 100, M, 0, scale=scale)
    want, tol = attend64(q, kc, vc, tables, lens, scale, 0)
    close(got, want, tol)


def test_attention_peaked_weights_and_flat_ones(zh, ctx):
    """One token takes everything / every token alike, over parts and steps."""
    rng = np.random.default_rng(7)
    P, lens = 1000, [1300, 1001, 1200]
    kc, vc, tables, _, M = make(rng, 3, 1, 128, P, lens)
    q = rng.standard_normal((3, 2, 128)).astype(np.float32)
    for where in (3, 999, 1000):
        k2 = kc.copy()
        slot = int(tables[0, where // 16]) * 16 + where % 16
        k2[0, slot] = (q[0, 0] * 3).astype(np.float16)
        got = run_attention(zh, ctx, q, k2, vc, tables, lens, P, M, 0)
        want, tol = attend64(q, k2, vc, tables, lens, 128 ** -0.5, 0, P)
        close(got, want, tol)
    q[:] = 0
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 0)
    want, tol = attend64(q, kc, vc, tables, lens, 128 ** -0.5, 0, P)
    close(got, want, tol)


def test_attention_nan_and_inf_stay_in_their_rows(zh, ctx):
    """A NaN of one sequence's own token, or of one query, is no other row's."""
    rng = np.random.default_rng(8)
    P, lens = 96, [130, 97, 160, 40]
    kc, vc, tables, _, M = make(rng, 4, 2, 128, P, lens)
    q = rng.standard_normal((4, 8, 128)).astype(np.float32)
    vc[1, int(tables[2, 150 // 16]) * 16 + 150 % 16, 5] = np.inf  # sequence 2, kv head 1, dim 5
    q[0, 3, 7] = np.nan
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 0)
    ok = np.ones(got.shape, bool)
    ok[2, 4:, 5] = False
    ok[0, 3] = False
    assert np.isnan(got[0, 3]).all() and not np.isfinite(got[2, 4:, 5]).any()
    qq = q.copy()
    qq[0, 3, 7] = 0
    vc = np.where(np.isinf(vc), np.float16(0), vc)
    want, tol = attend64(qq, kc, vc, tables, lens, 128 ** -0.5, 0)
    close(got, want, tol, ok)


def test_attention_cuts_lengths_and_reads_outside_pages_as_page_0(zh, ctx):
    rng = np.random.default_rng(10)
    lens = [64, 50]
    kc, vc, tables, _, M = make(rng, 2, 1, 64, 0, lens, poison=False)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    got = run_attention(zh, ctx, q, kc, vc, tables, [64, 5000], 0, 50, 0, expect_error=True)
    want, tol = attend64(q, kc, vc, tables, [50, 50], 0.125, 0)
    close(got, want, tol)
    for entry in (kc.shape[1] // 16, 0x10000000, 0xFFFFFFFF):
        bad = tables.copy()
        bad[1, 2] = entry
        got = run_attention(zh, ctx, q, kc, vc, bad, lens, 0, M, 0, expect_error=True)
        bad[1, 2] = 0
        want, tol = attend64(q, kc, vc, bad, lens, 0.125, 0)
        close(got, want, tol)


def test_attention_like_one_sequence_at_a_time(zh, ctx):
    """zh_flash_decode of each sequence: the same softmax within both bounds."""
    rng = np.random.default_rng(11)
    P, lens = 512, [700, 513, 612]
    kc, vc, tables, tokens, M = make(rng, 3, 8, 128, P, lens, poison=False)
    tables[tables == 0xFFFFFFF0] = 0
    q = rng.standard_normal((3, 32, 128)).astype(np.float32)
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 0)
    _, tol = attend64(q, kc, vc, tables, lens, 128 ** -0.5, 0)
    u = ctx.upload
    K, V, out = u(kc), u(vc), ctx.alloc(4 * 32 * 128)
    for s, n in enumerate(lens):
        ctx.flash_decode(u(q[s]), K, V, u(tables[s]), tables.shape[1], tokens, out, 32, 8, 128, n)
        one = out.download(np.float32, 32 * 128).reshape(32, 128)
        assert (np.abs(got[s] - one) <= 2 * tol[s]).all()


def test_two_contexts_at_once(zh, ctx):
    """Two contexts (streams), driven by two host threads over the same caches,
    tables and queries, each with its own workspace and results."""
    import threading
    rng = np.random.default_rng(31)
    P, lens = 700, [701 + 40 * i for i in range(12)]
    kc, vc, tables, tokens, M = make(rng, 12, 4, 128, P, lens)
    q = rng.standard_normal((12, 16, 128)).astype(np.float32)
    want, tol = attend64(q, kc, vc, tables, lens, 128 ** -0.5, 0, P, [0, 5, 11])
    u = ctx.upload
    K, V, T, Q, L = u(kc), u(vc), u(tables), u(q), u(np.array(lens, np.uint32))
    got, failed = [None, None], []

    def work(i):
        try:
            with zh.Context(0) as c:
                kv = zh.KvBatch(K, V, T, 12, tables.shape[1], tokens, 4, 128)
                out, ws = c.alloc(q.nbytes), c.alloc(c.flash_decode_shared_ws(kv, 16, P, M))
                rows = zh.DecodeRows(q=Q, out=out, seq_lens=L, ws=ws, n_heads=16, prefix_len=P, max_len=M)
                for _ in range(50):
                    c.flash_decode_shared(kv, rows)
                c.sync()
                got[i] = out.download(np.float32, q.size).reshape(q.shape)
        except Exception as e:  # noqa: BLE001 (shown by the assertion)
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    assert np.array_equal(got[0], got[1])
    close(got[0][[0, 5, 11]].astype(np.float64), want[[0, 5, 11]], tol[[0, 5, 11]])


# ---------------------------------------------------------------------------
# together: a pool, a prompt, forks, copies and decode steps
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
def test_fork_and_decode_together(zh, ctx, t):
    """A prompt written in one call, forked five ways (copy on write of the page
    it ends in), decoded some steps, one branch dropped, the pool compacted, and
    decoded on: every step's attention against the formula over the K and V rows
    of each branch, kept in 64 bits on the host."""
    rng = np.random.default_rng(12)
    nh, nkv, hd, pool_pages, P = 8, 2, 128, 64, 75
    G = nh // nkv
    pool = zh.KvPagePool(pool_pages)
    tokens = pool_pages * 16
    u = ctx.upload
    kcb, vcb = (u(np.full((nkv, tokens, hd), np.nan, np.float16)) for _ in range(2))
    caches = zh.KvCaches([kcb, vcb], tokens, nkv, hd)
    freq = (1e4 ** (-np.arange(0, hd, 2) / hd)).astype(np.float32)
    qw, kw = ((1 + 0.1 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2))
    F, QW, KW = u(freq), u(qw), u(kw)
    stride = 12
    history = {}  # request -> (K rows 64 bit, K tolerance, V rows)

    def step(requests, positions, n_per):
        """Writes n_per rows of each request at its next positions; returns q."""
        T = len(requests) * n_per
        x = rng.standard_normal((T, nh + 2 * nkv, hd)).astype(np.float32)
        pos = np.concatenate([p + np.arange(n_per) for p in positions])
        tables = np.zeros((len(requests), stride), np.uint32)
        for i, r in enumerate(requests):
            pg = pool.pages(r)
            tables[i, :pg.size] = pg
        X, out = u(x), ctx.alloc(T * nh * hd * (4 if t == 0 else 2))
        TB = u(tables)
        kv = zh.KvBatch(kcb, vcb, TB, len(requests), stride, tokens, nkv, hd)
        w = (nh + 2 * nkv) * hd
        ctx.qk_norm_rope_kv_write_batched(kv, zh.QkvRows(
            q=X, k=X, v=X, k_off=4 * nh * hd, v_off=4 * (nh + nkv) * hd, q_stride=w, k_stride=w, v_stride=w, q_out=out,
            q_out_type=t, pos=u(pos.astype(np.uint32)), seq=u(np.repeat(np.arange(len(requests)), n_per).astype(np.uint32)),
            n_rows=T, n_q_heads=nh, rope_dim=hd, inv_freq=F, q_norm_w=QW, k_norm_w=KW))
        k64, mag = rope64(x[:, nh:nh + nkv], kw, freq, pos, 1e-6, hd)
        for i, r in enumerate(requests):
            k, kt, v = history.setdefault(r, ([], [], []))
            for j in range(n_per):
                k.append(k64[i * n_per + j])
                kt.append(mag[i * n_per + j] * 2.0 ** -19 + store_error(1, k64[i * n_per + j]))
                v.append(x[i * n_per + j, nh + nkv:].astype(np.float16).astype(np.float64))
        return kv, out, tables

    def attention(requests, kv, q, prefix):
        lens = [len(history[r][0]) for r in requests]
        n = ctx.flash_decode_shared_ws(kv, nh, prefix, stride * 16)
        out = ctx.alloc(len(requests) * nh * hd * 4)
        ctx.flash_decode_shared(kv, zh.DecodeRows(q=q, out=out, seq_lens=u(np.array(lens, np.uint32)), ws=ctx.alloc(n),
                                                  n_heads=nh, prefix_len=prefix, max_len=stride * 16, type=t))
        ctx.sync()
        got = out.download(NP_TYPE[t], len(requests) * nh * hd).reshape(-1, nh, hd).astype(np.float64)
        qs = q.download(NP_TYPE[t], len(requests) * nh * hd).reshape(-1, nh, hd).astype(np.float64)
        for i, r in enumerate(requests):
            K, KT, V = (np.array(a) for a in history[r])
            for h in range(nh):
                sc = K[:, h // G] @ qs[i, h] * hd ** -0.5
                # the cache holds K rounded: a score moves by at most d
                d = (KT[:, h // G] @ np.abs(qs[i, h])).max() * hd ** -0.5
                A = 1.45 * hd ** -0.5 * (np.abs(K[:, h // G]) @ np.abs(qs[i, h])).max()
                w = np.exp(sc - sc.max())
                w /= w.sum()
                W = w @ np.abs(V[:, h // G])
                want = w @ V[:, h // G]
                tol = W * (2 * np.expm1(2 * d) + 2.0 ** -17 * A + (len(sc) / 32 + 80) * 2.0 ** -23 +
                           (2.0 ** -11 if t else 0)) + store_error(t, want)
                assert (np.abs(got[i, h] - want) <= tol).all(), (r, h)

    pool.alloc_pages(0, -(-P // 16))
    step([0], [0], P)
    requests = [0, 1, 2, 3, 4, 5]
    for c in requests[1:]:
        pool.fork(0, c, -(-P // 16))
        history[c] = tuple(list(a) for a in history[0])
    for it in range(25):
        if it == 12:  # a branch ends, the pool is compacted
            pool.free_pages(3)
            requests.remove(3)
            src, dst = pool.compact()
            ctx.kv_copy_pages(caches, caches, dst, src)
            assert len(src)
        moves = []
        for r in requests:
            n = len(history[r][0])
            if n % 16 == 0:
                pool.alloc_pages(r, 1)
            else:
                s, d = pool.unshare(r, n // 16)
                if s != d:
                    moves.append((d, s))
        if moves:
            ctx.kv_copy_pages(caches, caches, [m[0] for m in moves], [m[1] for m in moves])
            assert it == 0
        kv, q, _ = step(requests, [len(history[r][0]) for r in requests], 1)
        attention(requests, kv, q, P if it % 2 else P // 16 * 16)


def test_engine_fork_kv(zh, ctx):
    """A prompt prefilled by one engine and forked into two of its context and
    one of another context decodes like engines that prefilled it themselves."""
    cfg = dict(n_layers=2, hidden=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn=1024, vocab=1000, n_experts=0,
               n_experts_used=0, expert_ffn=0, max_ctx=128, type_attn=12, type_ffn_gate_up=12, type_ffn_down=14,
               type_lm_head=14, type_embd=12, type_router=8, rope_base=1e6, eps=1e-6, seed=5)
    prompt = np.random.default_rng(3).integers(0, 1000, 37)
    base = zh.InferenceEngine(ctx, cfg)
    ctx2 = zh.Context(0)
    engines = [base, base.share(ctx), base.share(ctx), base.share(ctx2, 64)]
    order = np.random.default_rng(1).permutation(8).astype(np.uint32)
    engines[2].set_pages(order)
    base.prefill(prompt)
    for e in engines[1:]:
        e.fork_kv(base, 37)
    want = [base.read_kv(l, w, 0, 37) for l in range(2) for w in range(2)]
    for e in engines[1:]:
        for i, x in enumerate(want):
            assert np.array_equal(e.read_kv(i // 2, i % 2, 0, 37), x)
    toks = [e.generate([7], 6, start_pos=37) for e in engines]
    assert toks[1] == toks[0] and toks[2] == toks[0] and toks[3] == toks[0]
    for e, n, name in ((base, 5, "InvalidArgument"), (engines[3], 65, "ContextLengthExceeded")):
        with pytest.raises(zh.ZincError) as err:
            e.fork_kv(base, n)
        assert err.value.name == name
    engines[1].fork_kv(base, 0)
    for e in reversed(engines):
        e.deinit()
    ctx2.close()


def test_rope_of_more_rows_than_a_grid_is_high(zh, ctx):
    """70000 rows without a sequence list, head_dim 2 (the kernel for any shape
    takes at most 65535 rows a launch): row t is sequence t."""
    rng = np.random.default_rng(13)
    T, hd = 70000, 2
    x = rng.standard_normal((T, 3, hd)).astype(np.float32)
    pos = rng.integers(0, 16, T).astype(np.uint32)
    pages = rng.permutation(T).astype(np.uint32)
    freq = np.ones(1, np.float32)
    u = ctx.upload
    kc, vc, out = u(np.zeros((T * 16, hd), np.float16)), u(np.zeros((T * 16, hd), np.float16)), ctx.alloc(4 * T * hd)
    X = u(x)
    kv = zh.KvBatch(kc, vc, u(pages), T, 1, T * 16, 1, hd)
    ctx.qk_norm_rope_kv_write_batched(kv, zh.QkvRows(
        q=X, k=X, v=X, k_off=4 * hd, v_off=8 * hd, q_stride=3 * hd, k_stride=3 * hd, v_stride=3 * hd, q_out=out,
        pos=u(pos), n_rows=T, n_q_heads=1, rope_dim=hd, inv_freq=u(freq)))
    ctx.sync()
    want, mag = rope64(x[:, :2], None, freq, pos, 1e-6, hd)
    close(out.download(np.float32, T * hd).reshape(T, hd), want[:, 0], mag[:, 0] * 2.0 ** -19)
    slot = pages.astype(np.int64) * 16 + pos
    k64 = np.zeros((T * 16, hd))
    k64[slot] = want[:, 1]
    v64 = np.zeros((T * 16, hd))
    v64[slot] = x[:, 2].astype(np.float16)
    close(kc.download(np.float16, k64.size).reshape(k64.shape), k64, 2.0 ** -19 * 2 * np.abs(k64).max() + store_error(1, k64))
    assert np.array_equal(vc.download(np.float16, v64.size).reshape(v64.shape).astype(np.float64), v64)


def test_rope_of_more_rows_than_a_launch_has(zh, ctx):
    """2^23 + 5 rows of head_dim 64 (a launch takes 2^23), all but the first and
    the last three padded, without a sequence list and with one."""
    rng = np.random.default_rng(14)
    T, hd, w = (1 << 23) + 5, 64, 192
    at = [0, T - 3, T - 2, T - 1]
    x = rng.standard_normal((4, 3, hd)).astype(np.float16)
    pos = np.full(T, NONE, np.uint32)
    pos[at] = [3, 15, 0, 7]
    u = ctx.upload
    X, P = ctx.alloc(2 * T * w), u(pos)
    seq = np.zeros(T, np.uint32)
    seq[at] = [0, 1, 2, 3]
    S = u(seq)
    for listed in (False, True):
        n_seq, of = (4, [0, 1, 2, 3]) if listed else (T, at)
        table = np.full(n_seq, 4, np.uint32)  # (outside the cache)
        table[of] = [2, 0, 3, 1]
        kc, vc = (u(np.zeros((64, hd), np.float16)) for _ in range(2))
        for r, row in zip(at, x):
            X.upload(row, 2 * r * w)
        kv = zh.KvBatch(kc, vc, u(table), n_seq, 1, 64, 1, hd)
        ctx.qk_norm_rope_kv_write_batched(kv, zh.QkvRows(
            q=X, k=X, v=X, k_off=2 * hd, v_off=4 * hd, q_stride=w, k_stride=w, v_stride=w, q_out=X, q_out_stride=w,
            pos=P, seq=S if listed else None, n_rows=T, n_q_heads=1, type=1, rope_dim=hd, inv_freq=u(np.ones(hd // 2, np.float32))))
        ctx.sync()
        want, mag = rope64(x[:, :2].astype(np.float64), None, np.ones(hd // 2, np.float32), pos[at], 1e-6, hd)
        got = np.stack([X.download(np.float16, hd, 2 * r * w) for r in at])
        close(got, want[:, 0], mag[:, 0] * 2.0 ** -19 + store_error(1, want[:, 0]))
        k64, v64, tol = np.zeros((64, hd)), np.zeros((64, hd)), np.zeros((64, hd))
        slot = np.array([2, 0, 3, 1]) * 16 + pos[at]
        k64[slot], v64[slot] = want[:, 1], x[:, 2]
        tol[slot] = mag[:, 1] * 2.0 ** -19
        close(kc.download(np.float16, k64.size).reshape(k64.shape), k64, tol + store_error(1, k64))
        assert np.array_equal(vc.download(np.float16, v64.size).reshape(v64.shape).astype(np.float64), v64)


def test_engine_fork_kv_then_a_batch(zh, ctx):
    """A prompt prefilled once and forked into the engines of a decode batch
    gives each the tokens of its own continuation; a page table that names a
    page twice is refused."""
    cfg = dict(n_layers=2, hidden=512, n_heads=4, n_kv_heads=2, head_dim=128, ffn=1024, vocab=1000, n_experts=0,
               n_experts_used=0, expert_ffn=0, max_ctx=128, type_attn=12, type_ffn_gate_up=12, type_ffn_down=14,
               type_lm_head=14, type_embd=12, type_router=8, rope_base=1e6, eps=1e-6, seed=5)
    prompt = np.random.default_rng(4).integers(0, 1000, 50)
    base = zh.InferenceEngine(ctx, cfg)
    engines = [base] + [base.share(ctx) for _ in range(3)]
    base.prefill(prompt)
    for e in engines[1:]:
        e.fork_kv(base, 50)
    starts = [[3], [500], [77], [999]]
    want = [e.generate(p, 5, start_pos=50) for e, p in zip(engines, starts)]
    assert zh.InferenceEngine.generate_batch(engines, starts, 5, start_pos=50) == want
    engines[3].set_pages(np.zeros(8, dtype=np.uint32))
    with pytest.raises(zh.ZincError) as err:
        engines[3].fork_kv(base, 50)
    assert err.value.name == "InvalidArgument"
    engines[3].fork_kv(base, 16)
    for e in reversed(engines):
        e.deinit()

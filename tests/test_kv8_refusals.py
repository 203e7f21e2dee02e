"""What the operators over an 8-bit cache refuse, host side (no GPU): the library's
own checks, over buffers that only look like device ones."""
import ctypes as C

import numpy as np
import pytest
from test_kv_batch import INVALID, OK, TOO_LONG, UNSUPPORTED, Fake, check
from test_kv_batch_refusals import Owned, no_device_free, owned  # noqa: F401 (a fixture)

import zinc_amd
from zinc_amd import E4M3, F16, F32, I8, AttnRows, Kv8Batch, Kv8Caches, KvCaches, QkvRows, hip

NKV, HD, TOKENS, SEQS, STRIDE, CUS = 2, 128, 512, 5, 8, 256


def batch(**over):
    f = dict(k_cache=Fake(NKV * HD * TOKENS), v_cache=Fake(NKV * HD * TOKENS), k_scale=Fake(NKV * TOKENS // 4),
             v_scale=Fake(NKV * TOKENS // 4), tables=Fake(4 * SEQS * STRIDE), seq_lens=Fake(4 * SEQS), n_seq=SEQS,
             table_stride=STRIDE, cache_tokens=TOKENS, n_kv_heads=NKV, head_dim=HD, type=I8)
    f.update(over)
    return Kv8Batch(**f)


def qkv(n=4, nq=6, **over):
    f = dict(q=Fake(4 * n * nq * HD), k=Fake(4 * n * NKV * HD), v=Fake(4 * n * NKV * HD), q_out=Fake(4 * n * nq * HD),
             pos=None, n_rows=n, n_q_heads=nq, inv_freq=Fake(2 * HD), rope_dim=HD)
    f.update(over)
    return QkvRows(**f)


def attn(n=4, nh=6, **over):
    f = dict(q=Fake(4 * n * nh * HD), out=Fake(4 * n * nh * HD), ws=Fake(1 << 28), n_rows=n, max_rows=1, max_len=128,
             n_heads=nh)
    f.update(over)
    return AttnRows(**f)


def write_check(kv, r):
    return check("zh_check_kv8_rows", kv.ptr, r.ptr)


def attn_check(kv, r):
    return check("zh_check_attn_kv8", kv.ptr, r.ptr, C.c_uint32(CUS))


def ws_bytes(kv, n_heads, n_rows, max_rows, max_len):
    f = zinc_amd.lib().zh_check_attn_kv8_ws
    f.restype = C.c_uint64
    return f(kv.ptr, *[C.c_uint32(x) for x in (n_heads, n_rows, max_rows, max_len, CUS)])


BAD_BATCHES = [dict(n_seq=0), dict(table_stride=0), dict(cache_tokens=0), dict(cache_tokens=500), dict(n_kv_heads=0),
               dict(head_dim=0), dict(head_dim=96), dict(head_dim=256), dict(n_seq=6), dict(table_stride=9),
               dict(cache_tokens=528), dict(k_cache=None), dict(tables=None), dict(seq_lens=None), dict(v_scale=None),
               dict(v_cache=Fake(NKV * HD * TOKENS - 1)), dict(k_scale=Fake(NKV * TOKENS // 4 - 4)),
               dict(seq_lens=Fake(4 * SEQS - 4)), dict(row_start=Fake(4 * SEQS))]


@pytest.mark.parametrize("over", BAD_BATCHES, ids=lambda o: next(iter(o)))
def test_bad_batches(over):
    assert write_check(batch(**over), qkv()) == INVALID
    assert attn_check(batch(**over), attn()) == INVALID
    assert ws_bytes(batch(**over), 6, 4, 1, 128) == 0


def test_batches_accepted():
    for kv in (batch(), batch(type=E4M3), batch(row_start=Fake(4 * SEQS + 4))):
        assert write_check(kv, qkv()) == OK and attn_check(kv, attn()) == OK
    assert write_check(batch(), qkv(n=6)) == INVALID and attn_check(batch(), attn(n=6)) == INVALID  # a row without a sequence
    kv = batch(row_start=Fake(4 * SEQS + 4))
    assert write_check(kv, qkv(n=60)) == OK and attn_check(kv, attn(n=60, max_rows=60)) == OK
    for t in (F32, F16, 8, 0x18 + 1):
        assert write_check(batch(type=t), qkv()) == UNSUPPORTED and attn_check(batch(type=t), attn()) == UNSUPPORTED


def test_one_buffer_in_two_places():
    one = Fake(1 << 20)
    names = ["k_cache", "v_cache", "k_scale", "v_scale"]
    for i, a in enumerate(names):
        for b in names[:i] + ["tables", "seq_lens", "row_start"]:
            kv = batch(**{a: one, b: one})
            assert write_check(kv, qkv()) == INVALID and attn_check(kv, attn()) == INVALID
    for n in names + ["tables", "seq_lens", "row_start"]:
        kv = batch(**{n: one})
        assert write_check(kv, qkv(q_out=one)) == INVALID and attn_check(kv, attn(out=one)) == INVALID
        long = dict(table_stride=4096, max_len=60000)
        kv = batch(**{"tables": Fake(4 * SEQS * 4096), n: one}, table_stride=4096) if n != "tables" else batch(tables=one, table_stride=4096)
        assert attn_check(kv, attn(max_len=long["max_len"])) == OK
        assert attn_check(kv, attn(max_len=long["max_len"], ws=one)) == INVALID
    for n in names:
        for m in ("q", "k", "v", "inv_freq", "q_norm_w"):
            assert write_check(batch(**{n: one}), qkv(**{m: one})) == INVALID


@pytest.mark.parametrize("over", [
    dict(n_q_heads=0), dict(n_q_heads=5), dict(n_q_heads=8), dict(rope_dim=12), dict(rope_dim=136), dict(n_rows=5),
    dict(q_stride=6 * HD - 4), dict(q_stride=6 * HD + 2), dict(k_stride=NKV * HD + 1), dict(v_off=8), dict(q_off=4),
    dict(q_out_off=8), dict(inv_freq=None), dict(pos=Fake(16)), dict(seq=Fake(16)), dict(q_norm_w=Fake(4 * HD - 4)),
    dict(q_out=None), dict(k=None), dict(v_stride=1 << 31, n_rows=3)], ids=str)
def test_bad_rows(over):
    assert write_check(batch(), qkv(**over)) == INVALID


def test_rows_accepted():
    for r in (qkv(), qkv(n_rows=0), qkv(rope_dim=0, inv_freq=None), qkv(rope_dim=8), qkv(type=F16), qkv(q_out_type=F16)):
        assert write_check(batch(), r) == OK
    q = Fake(4 * 4 * 10 * HD)  # stacked rows q | k | v, q_out in place
    stacked = dict(q=q, k=q, v=q, k_off=4 * 6 * HD, v_off=4 * 8 * HD, q_stride=10 * HD, k_stride=10 * HD, v_stride=10 * HD)
    assert write_check(batch(), qkv(q_out=q, q_out_stride=10 * HD, **stacked)) == OK
    assert write_check(batch(), qkv(q_out=q, q_out_off=4 * HD, q_out_stride=10 * HD, **stacked)) == INVALID
    assert write_check(batch(), qkv(type=9)) == UNSUPPORTED


@pytest.mark.parametrize("over", [
    dict(n_heads=0), dict(n_heads=5), dict(n_heads=8), dict(n_rows=0), dict(max_rows=0), dict(max_rows=5),
    dict(max_len=0), dict(max_len=(1 << 30) + 1), dict(q_off=8), dict(out_off=4), dict(q_stride=6 * HD - 4),
    dict(out_stride=6 * HD + 2), dict(q_stride=1 << 31), dict(out=None), dict(q=None), dict(attn_scale=float("nan")),
    dict(attn_scale=float("-inf"))], ids=str)
def test_bad_attention(over):
    assert attn_check(batch(), attn(**over)) == INVALID


def test_attention_rest():
    assert attn_check(batch(), attn(max_len=129)) == TOO_LONG and attn_check(batch(), attn(type=8)) == UNSUPPORTED
    for r in (attn(attn_scale=-3.0), attn(type=F16), attn(ws=None), attn(n=1, q_stride=4, out_stride=4)):
        assert attn_check(batch(), r) == OK
    q = Fake(4 * 4 * 8 * HD)
    assert attn_check(batch(), attn(q=q, out=q)) == OK
    assert attn_check(batch(), attn(q=q, out=q, out_off=4 * HD)) == INVALID
    assert attn_check(batch(), attn(q=q, out=q, q_stride=7 * HD)) == INVALID
    wide = Fake(4 * 4 * 12 * HD)  # in the other columns of the same rows
    assert attn_check(batch(), attn(q=wide, out=wide, q_stride=12 * HD, out_stride=12 * HD, out_off=4 * 6 * HD)) == OK
    kv = batch(table_stride=4096, tables=Fake(4 * SEQS * 4096))
    for ws in (None, Fake(64)):
        assert attn_check(kv, attn(max_len=60000, ws=ws)) == INVALID
    for n in ("q", "out"):
        one = Fake(1 << 30)
        assert attn_check(kv, attn(max_len=60000, ws=one, **{n: one})) == INVALID


def test_launches_too_large():
    n = 1 << 22
    kv = batch(n_seq=n, table_stride=1, tables=Fake(4 * n), seq_lens=Fake(4 * n))
    big = dict(q=Fake(1 << 42), out=Fake(1 << 42), ws=Fake(1 << 45), max_len=16)
    assert attn_check(kv, attn(**big)) == INVALID
    kv = batch(n_seq=n - 1, table_stride=1, tables=Fake(4 * n), seq_lens=Fake(4 * n))
    assert attn_check(kv, attn(**big)) == OK
    rows = dict(n_rows=(1 << 30) - 1, max_rows=(1 << 30) - 1)
    kv = batch(row_start=Fake(4 * SEQS + 4))
    assert attn_check(kv, attn(**big, **rows)) == INVALID


NAMES = ["k_cache", "v_cache", "k_scale", "v_scale", "tables", "seq_lens", "row_start"]


@pytest.mark.parametrize("name", NAMES)
def test_a_batch_of_a_freed_buffer(no_device_free, name):  # noqa: F811
    kv, bufs = owned(batch, **{n: 1 << 20 for n in NAMES})
    assert write_check(kv, qkv()) == OK and attn_check(kv, attn()) == OK
    bufs[name].free()
    assert write_check(kv, qkv()) == INVALID and attn_check(kv, attn()) == INVALID and ws_bytes(kv, 6, 4, 1, 64) == 0


@pytest.mark.parametrize("name", ["q", "out", "ws"])
def test_attention_rows_of_a_freed_buffer(no_device_free, name):  # noqa: F811
    rows, bufs = owned(attn, **{n: 1 << 26 for n in ("q", "out", "ws")})
    assert attn_check(batch(), rows) == OK
    bufs[name].free()
    assert attn_check(batch(), rows) == INVALID


def test_a_workspace_serves_every_smaller_call():
    """Whatever is smaller in it, of either type: no call may be refused for its ws."""
    rng = np.random.default_rng(3)
    some = lambda top: int(min(top, np.exp(rng.uniform(0, np.log(top + 1)))))  # noqa: E731
    asked = 0
    for _ in range(400):
        nkv, hd = int(rng.choice([1, 2, 4, 8])), int(rng.choice([64, 128]))
        G, n_seq, max_len = int(rng.choice([1, 2, 4, 5, 8, 16])), some(300), some(200000)
        rows = some(4000)
        n_rows = min(rows * some(n_seq), 20000)
        rows = min(rows, n_rows)
        kv = lambda n: Kv8Batch(*[Fake(1 << 30) for _ in range(6)], row_start=Fake(1 << 20), n_seq=n, table_stride=12500,  # noqa: E731
                                cache_tokens=16, n_kv_heads=nkv, head_dim=hd, type=I8)
        size = ws_bytes(kv(n_seq), G * nkv, n_rows, rows, max_len)
        if size == 0:
            continue
        for _ in range(12):
            less = [x if rng.integers(2) else some(x) for x in (n_seq, n_rows, rows, max_len)]
            r = AttnRows(q=Fake(1 << 40), out=Fake(1 << 40), ws=Fake(size), n_rows=less[1], max_rows=min(less[1:3]),
                         max_len=less[3], n_heads=G * nkv, type=int(rng.integers(2)))
            assert attn_check(kv(less[0]), r) == OK, (nkv, hd, G, n_seq, n_rows, rows, max_len, less)
            asked += 1
    assert asked > 3000
    assert size < 1 << 30


# ---- pages
def pages_check(op, dst, src, dp, sp, n=None):
    d, s = np.array(dp, dtype=np.uint32), np.array(sp, dtype=np.uint32)
    dst8, src8 = (dst if op != 1 else None), (src if op != 0 else None)
    half = src if op == 0 else dst if op == 1 else None
    return check("zh_check_kv8_pages", C.c_uint32(op), dst8 and dst8.ptr, src8 and src8.ptr, half and half.ptr,
                 C.c_void_p(d.ctypes.data), C.c_void_p(s.ctypes.data), C.c_uint32(len(d) if n is None else n))


def set8(n=2, tokens=160, nkv=2, hd=64, t=I8, bufs=None, scales=None):
    return Kv8Caches(bufs or [Fake(nkv * hd * tokens) for _ in range(n)],
                     scales or [Fake(nkv * tokens // 4) for _ in range(n)], tokens, nkv, hd, t)


def set16(n=2, tokens=160, nkv=2, hd=64, bufs=None):
    return KvCaches(bufs or [Fake(2 * nkv * hd * tokens) for _ in range(n)], tokens, nkv, hd)


def test_pages_accepted():
    a, b, h = set8(), set8(tokens=320), set16(tokens=480)
    assert pages_check(0, a, h, [9, 0], [29, 29]) == OK      # a source page twice
    assert pages_check(1, h, a, [29, 3], [0, 0]) == OK
    assert pages_check(2, b, a, [19, 9], [9, 9]) == OK
    assert pages_check(2, a, a, [1, 2, 3], [4, 5, 4]) == OK
    for op, x, y in ((0, a, h), (1, h, a), (2, a, b), (2, a, a)):
        assert pages_check(op, x, y, [], []) == OK


def test_pages_refused():
    a, b, h = set8(), set8(tokens=320), set16(tokens=480)
    for op, x, y, dn, sn in ((0, a, h, 10, 30), (1, h, a, 30, 10), (2, b, a, 20, 10)):
        assert pages_check(op, x, y, [dn], [0]) == INVALID and pages_check(op, x, y, [0], [sn]) == INVALID
        assert pages_check(op, x, y, [3, 1, 3], [1, 2, 3]) == INVALID   # two to one page
        assert check("zh_check_kv8_pages", C.c_uint32(op), a.ptr, a.ptr, h.ptr, None, None, C.c_uint32(1)) == INVALID
    assert pages_check(2, a, a, [1, 2], [2, 5]) == INVALID               # page 2 read and written
    for other in (dict(n=3), dict(nkv=4), dict(hd=128)):
        for op, x, y in ((0, set8(**other), h), (1, h, set8(**other)), (2, a, set8(**other)), (0, a, set16(**other))):
            assert pages_check(op, x, y, [1], [2]) == INVALID
    assert pages_check(2, a, set8(t=E4M3), [1], [2]) == INVALID          # codes of another type
    assert pages_check(0, set8(t=F16), h, [1], [2]) == UNSUPPORTED
    for bad in (dict(n=257), dict(tokens=168), dict(hd=96)):
        assert pages_check(2, set8(**bad), set8(**bad), [1], [2]) == INVALID
    assert pages_check(2, set8(n=256), set8(n=256), [1], [2]) == OK
    small = [Fake(2 * 64 * 160), Fake(2 * 64 * 160 - 1)]
    assert pages_check(2, set8(bufs=small), a, [1], [2]) == INVALID
    assert pages_check(2, a, set8(scales=[Fake(80), Fake(76)]), [1], [2]) == INVALID
    one, two = Fake(1 << 20), Fake(1 << 20)
    assert pages_check(0, set8(bufs=[one, one]), h, [1], [2]) == INVALID
    assert pages_check(0, set8(bufs=[one, two], scales=[Fake(80), one]), h, [1], [2]) == INVALID
    assert pages_check(0, set8(bufs=[one, two]), set16(bufs=[two, Fake(1 << 20)]), [1], [2]) == INVALID
    assert pages_check(2, set8(bufs=[one, two]), set8(bufs=[two, one]), [1], [2]) == INVALID


def test_a_set_of_a_freed_buffer(no_device_free):  # noqa: F811
    for which in range(4):
        bufs = [Owned(1 << 20) for _ in range(4)]
        a = Kv8Caches(bufs[:2], bufs[2:], 64, 1, 64, I8)
        assert pages_check(2, a, a, [1], [2]) == OK
        bufs[which].free()
        assert pages_check(2, a, a, [1], [2]) == INVALID


def test_python_refusals():
    with pytest.raises(ValueError):
        Kv8Caches([Fake(1 << 20)], [], 64, 1, 64, I8)
    a, h = set8(), set16()

    class Methods:  # of a Context, without a device
        h = None
        _kv8_pages, unpack = hip.Context._kv8_pages, hip.Context.kv8_unpack_pages
        pack, copy = hip.Context.kv8_pack_pages, hip.Context.kv8_copy_pages

    c = Methods()
    for f, x, y in ((c.unpack, h, a), (c.copy, a, a)):
        with pytest.raises(ValueError):
            f(x, y, [1, 2], [3])
    for dp, sp, n in (([1, 2], [3, 4], 16), ([1], [3, 4], 16), ([], [], -5), ([1], [2], 0), ([1], [2], (1 << 32) + 16)):
        with pytest.raises(ValueError):
            c.pack(a, h, dp, sp, n)


def test_entries_refuse_a_null_context():
    L = zinc_amd.lib()
    a, h, p = set8(), set16(), np.zeros(1, dtype=np.uint32).ctypes.data
    assert L.zh_qk_norm_rope_kv8_write_batched(None, batch().ptr, qkv().ptr) == INVALID
    assert L.zh_flash_attn_kv8(None, batch().ptr, attn().ptr) == INVALID
    assert L.zh_flash_attn_kv8_ws(None, batch().ptr, 6, 4, 1, 128) == 0
    assert L.zh_kv8_pack_pages(None, a.ptr, h.ptr, p, p, 0) == INVALID
    assert L.zh_kv8_unpack_pages(None, h.ptr, a.ptr, p, p, 0) == INVALID
    assert L.zh_kv8_copy_pages(None, a.ptr, a.ptr, p, p, 0) == INVALID

"""The batched operators over a paged KV cache, host side (no GPU): sharing,
trimming and compacting the pages of the pool, and every refusal of
zh_kv_copy_pages, zh_qk_norm_rope_kv_write_batched and zh_flash_decode_shared
(the library's own checks, over buffers that only look like device ones)."""
import ctypes as C

import numpy as np
import pytest

import zinc_amd
from zinc_amd import F16, F32, KvBatch, KvCaches, KvPagePool, ZincError, hip
from zinc_amd.hip import DecodeRows, QkvRows

OK, UNSUPPORTED, INVALID, TOO_LONG = 0, 1, 2, 4


# ---- pool
def test_fork_shares_and_frees_with_the_last_holder():
    pool = KvPagePool(8, 16)
    a = pool.alloc_pages(1, 4)
    pool.fork(1, 2, 3)
    pool.fork(1, 3, 4)
    assert pool.pages(2).tolist() == a[:3].tolist() and pool.free_count() == 4
    assert [pool.refs(p) for p in a] == [3, 3, 3, 2]
    pool.free_pages(1)
    assert pool.free_count() == 4 and pool.pages(1).size == 0
    pool.free_pages(3)
    assert pool.free_count() == 5 and [pool.refs(p) for p in a] == [1, 1, 1, 0]
    pool.free_pages(2)
    assert pool.free_count() == 8
    pool.free_pages(2)
    assert pool.free_count() == 8


def test_fork_refusals():
    pool = KvPagePool(8, 16)
    pool.alloc_pages(1, 2)
    pool.alloc_pages(2, 1)
    for args in ((1, 2, 1), (1, 1, 1), (1, 3, 3), (9, 3, 1)):  # child with pages, itself, too many, no parent
        with pytest.raises(ZincError) as e:
            pool.fork(*args)
        assert e.value.name == "InvalidArgument"
    pool.fork(1, 3, 0)
    assert pool.pages(3).size == 0 and pool.free_count() == 5


def test_unshare_replaces_a_shared_page_only():
    pool = KvPagePool(4, 16)
    a = pool.alloc_pages(1, 2)
    pool.fork(1, 2, 2)
    src, dst = pool.unshare(2, 1)
    assert src == a[1] and dst not in a and pool.pages(2).tolist() == [a[0], dst]
    assert pool.pages(1).tolist() == a.tolist() and pool.refs(src) == 1 and pool.refs(dst) == 1
    assert pool.unshare(2, 1) == (dst, dst) and pool.unshare(1, 1) == (a[1], a[1])
    pool.alloc_pages(3, 1)
    with pytest.raises(ZincError) as e:
        pool.unshare(1, 0)
    assert e.value.name == "KvCacheExhausted" and pool.pages(1).tolist() == a.tolist()
    for r, i in ((1, 2), (7, 0)):
        with pytest.raises(ZincError) as e:
            pool.unshare(r, i)
        assert e.value.name == "InvalidArgument"


def test_trim():
    pool = KvPagePool(8, 16)
    a = pool.alloc_pages(1, 5)
    pool.fork(1, 2, 3)
    pool.trim(1, 2)
    assert pool.pages(1).tolist() == a[:2].tolist() and pool.free_count() == 5 and pool.refs(a[2]) == 1
    pool.trim(1, 2)
    pool.trim(5, 0)
    pool.trim(1, 0)
    assert pool.pages(1).size == 0 and pool.free_count() == 5
    pool.free_pages(2)
    assert pool.free_count() == 8


def test_compact_moves_the_pages_in_use_down():
    pool = KvPagePool(10, 16)
    for r in range(5):
        pool.alloc_pages(r, 2)  # 9 8 | 7 6 | 5 4 | 3 2 | 1 0
    pool.fork(1, 9, 2)
    pool.free_pages(4)
    pool.free_pages(2)  # free: 0 1 4 5, in use 2 3 6 7 8 9
    before = {r: pool.pages(r) for r in (0, 1, 3, 9)}
    src, dst = pool.compact()
    assert sorted(src.tolist()) == [6, 7, 8, 9] and sorted(dst.tolist()) == [0, 1, 4, 5]
    to = dict(zip(src.tolist(), dst.tolist()))
    for r, p in before.items():
        assert pool.pages(r).tolist() == [to.get(x, x) for x in p.tolist()]
    assert pool.refs(to[7]) == 2 and pool.refs(7) == 0 and pool.free_count() == 4
    assert pool.compact()[0].size == 0
    assert pool.alloc_pages(20, 4).tolist() == [9, 8, 7, 6]
    with pytest.raises(ZincError):
        pool.alloc_pages(21, 1)


def test_compact_refuses_short_arrays_and_changes_nothing():
    pool = KvPagePool(6, 16)
    a = pool.alloc_pages(1, 3)
    n, one = C.c_uint32(), np.empty(1, dtype=np.uint32)
    rc = zinc_amd.lib().zh_kv_pool_compact(pool.h, one.ctypes.data, one.ctypes.data, 1, C.byref(n))
    assert rc == INVALID and n.value == 3 and pool.pages(1).tolist() == a.tolist() and pool.free_count() == 3


def test_pool_random_against_a_model():
    rng = np.random.default_rng(5)
    total = 40
    pool, held = KvPagePool(total, 16), {}
    content = np.zeros(total, dtype=np.int64)  # what each page holds
    for step in range(600):
        op, r = rng.integers(6), int(rng.integers(12))
        if op == 0 and pool.free_count() >= 3:
            for p in pool.alloc_pages(r, int(rng.integers(1, 4))):
                content[p] = step * 100 + len(held.setdefault(r, []))
                held[r].append(content[p])
        elif op == 1:
            pool.free_pages(r)
            held.pop(r, None)
        elif op == 2:
            c = int(rng.integers(12))
            if held.get(r) and not held.get(c):
                n = int(rng.integers(1, len(held[r]) + 1))
                pool.fork(r, c, n)
                held[c] = held[r][:n]
        elif op == 3 and held.get(r) and pool.free_count():
            i = int(rng.integers(len(held[r])))
            src, dst = pool.unshare(r, i)
            content[dst] = content[src] if src == dst else step * 100 + 50
            held[r][i] = content[dst]
        elif op == 4:
            k = int(rng.integers(4))
            pool.trim(r, k)
            if r in held:
                held[r] = held[r][:k]
        elif op == 5:
            src, dst = pool.compact()
            content[dst] = content[src]
        pages = {q: pool.pages(q) for q in range(12)}
        for q in range(12):
            assert content[pages[q]].tolist() == held.get(q, [])
        used = np.concatenate(list(pages.values()))
        assert pool.free_count() == total - np.unique(used).size
        assert all(pool.refs(p) == np.sum(used == p) for p in range(total))


# ---- refusals
class FakeBuf(C.Structure):
    """A zh_buf as the host checks see it: an address and a size."""
    _fields_ = [("p", C.c_uint64), ("size", C.c_uint64)]


class Fake(hip.Buffer):
    at = 1 << 40

    def __init__(self, size, address=None):
        self._b = FakeBuf(Fake.at if address is None else address, size)
        Fake.at += (size + 4095) // 4096 * 4096 + 4096
        self.h, self.size = C.addressof(self._b), size

    def free(self):
        pass


def check(name, *args):
    f = getattr(zinc_amd.lib(), name)
    f.restype = C.c_int
    return f(None, *args)


def copy_check(dst, src, dp, sp):
    d, s = np.asarray(dp, dtype=np.uint32), np.asarray(sp, dtype=np.uint32)
    return check("zh_check_kv_copy_pages", dst.ptr, src.ptr, C.c_void_p(d.ctypes.data), C.c_void_p(s.ctypes.data),
                 C.c_uint32(len(d)))


def test_copy_refusals():
    nkv, hd, tokens = 2, 64, 160
    size = 2 * nkv * hd * tokens
    bufs = [Fake(size) for _ in range(4)]
    a, b = KvCaches(bufs[:2], tokens, nkv, hd), KvCaches(bufs[2:], tokens, nkv, hd)
    assert copy_check(a, a, [1, 2, 3], [4, 5, 4]) == OK
    assert copy_check(a, a, [], []) == OK
    assert copy_check(a, b, [1, 2], [2, 1]) == OK          # other caches: no page is both
    assert copy_check(a, a, [1, 2], [2, 5]) == INVALID     # page 2 read and written
    assert copy_check(a, a, [3], [3]) == INVALID
    assert copy_check(a, b, [1, 1], [2, 3]) == INVALID     # written twice
    assert copy_check(a, a, [10], [1]) == INVALID and copy_check(a, a, [1], [10]) == INVALID
    assert copy_check(a, a, [1], [0xFFFFFFFF]) == INVALID
    crossed = KvCaches([bufs[1], bufs[0]], tokens, nkv, hd)
    assert copy_check(a, crossed, [1, 2], [2, 3]) == INVALID
    assert copy_check(KvCaches([bufs[0]] * 2, tokens, nkv, hd), b, [1], [1]) == INVALID  # one cache twice
    assert copy_check(a, KvCaches(bufs[2:3], tokens, nkv, hd), [1], [1]) == INVALID
    assert copy_check(a, KvCaches(bufs[2:], tokens, 1, hd), [1], [1]) == INVALID
    assert copy_check(KvCaches(bufs[:2], tokens + 16, nkv, hd), b, [1], [1]) == INVALID  # past the buffers
    assert copy_check(KvCaches(bufs[:2], 150, nkv, hd), KvCaches(bufs[2:], 150, nkv, hd), [1], [1]) == INVALID
    assert copy_check(KvCaches([], tokens, nkv, hd), KvCaches([], tokens, nkv, hd), [1], [1]) == INVALID
    assert copy_check(KvCaches(bufs[:2], tokens // 2, nkv, hd), a, [1], [2]) == INVALID  # one cache in two sizes
    many = [Fake(4096) for _ in range(256)]
    assert copy_check(KvCaches(many, 16, 1, 64), KvCaches(many[::-1], 16, 1, 64), [0], [0]) == INVALID  # read and written
    assert copy_check(KvCaches(many, 16, 1, 64), KvCaches([Fake(4096) for _ in range(256)], 16, 1, 64), [0], [0]) == OK
    assert copy_check(KvCaches(many + bufs[:1], 16, 1, 64), KvCaches(many + bufs[:1], 16, 1, 64), [], []) == INVALID
    assert check("zh_check_kv_copy_pages", a.ptr, a.ptr, None, None, C.c_uint32(1)) == INVALID
    with pytest.raises(ValueError):
        hip.Context.kv_copy_pages(None, a, a, [1, 2], [3])


NKV, HD, TOKENS, SEQS, STRIDE = 2, 128, 512, 5, 8


def batch(**over):
    f = dict(k_cache=Fake(2 * NKV * HD * TOKENS), v_cache=Fake(2 * NKV * HD * TOKENS), tables=Fake(4 * SEQS * STRIDE),
             n_seq=SEQS, table_stride=STRIDE, cache_tokens=TOKENS, n_kv_heads=NKV, head_dim=HD)
    f.update(over)
    return KvBatch(**f)


BAD_BATCHES = [dict(n_seq=0), dict(table_stride=0), dict(cache_tokens=0), dict(cache_tokens=500), dict(n_kv_heads=0),
               dict(head_dim=0), dict(n_seq=6), dict(table_stride=9), dict(cache_tokens=528), dict(k_cache=None),
               dict(tables=None), dict(v_cache=Fake(2 * NKV * HD * TOKENS - 2))]


def qkv(n=4, nq=6, **over):
    f = dict(q=Fake(4 * n * nq * HD), k=Fake(4 * n * NKV * HD), v=Fake(4 * n * NKV * HD), q_out=Fake(4 * n * nq * HD),
             pos=Fake(4 * n), seq=Fake(4 * n), n_rows=n, n_q_heads=nq, inv_freq=Fake(2 * HD), rope_dim=HD)
    f.update(over)
    return QkvRows(**f)


def rows_check(kv, r):
    return check("zh_check_qkv_rows", kv.ptr, r.ptr)


def test_rows_accepted():
    kv = batch()
    for r in (qkv(), qkv(seq=None), qkv(n_rows=0), qkv(rope_dim=0, inv_freq=None), qkv(rope_dim=64), qkv(type=F16),
              qkv(q_out_type=F16), qkv(q_norm_w=Fake(4 * HD), k_norm_w=Fake(4 * HD))):
        assert rows_check(kv, r) == OK
    q = Fake(4 * 4 * 10 * HD)  # stacked rows q | k | v, q_out in place
    stacked = dict(q=q, k=q, v=q, k_off=4 * 6 * HD, v_off=4 * 8 * HD, q_stride=10 * HD, k_stride=10 * HD,
                   v_stride=10 * HD)
    assert rows_check(kv, qkv(**stacked)) == OK
    assert rows_check(kv, qkv(q_out=q, q_out_stride=10 * HD, **stacked)) == OK


@pytest.mark.parametrize("over", BAD_BATCHES, ids=lambda o: next(iter(o)))
def test_bad_batches(over):
    assert rows_check(batch(**over), qkv()) == INVALID
    assert check("zh_check_decode_rows", batch(**over).ptr, decode().ptr, C.c_uint32(256)) == INVALID


@pytest.mark.parametrize("over", [
    dict(n_q_heads=0), dict(n_q_heads=5), dict(n_q_heads=8), dict(rope_dim=63), dict(rope_dim=130), dict(n_rows=5),
    dict(q_stride=6 * HD - 1), dict(q_stride=6 * HD + 1), dict(k_stride=2 * HD - 1), dict(v_off=4), dict(q_off=2),
    dict(q_out_off=1), dict(inv_freq=None), dict(pos=None), dict(seq=Fake(12)), dict(q_norm_w=Fake(4 * HD - 4)),
    dict(q_out=None), dict(k=None)], ids=str)
def test_bad_rows(over):
    assert rows_check(batch(), qkv(**over)) == INVALID


def test_bad_rows_types_and_overlaps():
    assert rows_check(batch(), qkv(type=8)) == UNSUPPORTED and rows_check(batch(), qkv(q_out_type=8)) == UNSUPPORTED
    assert rows_check(batch(), qkv(n=6, seq=None)) == INVALID  # more rows than sequences
    q = Fake(4 * 4 * 10 * HD)
    assert rows_check(batch(), qkv(q=q, q_out=q)) == OK
    assert rows_check(batch(), qkv(q=q, q_out=q, q_out_off=4 * HD)) == INVALID
    assert rows_check(batch(), qkv(q=q, q_out=q, q_out_type=F16)) == INVALID
    assert rows_check(batch(), qkv(k=q, k_off=4 * HD, q_out=q)) == INVALID
    assert rows_check(batch(), qkv(v=q, q_out=q)) == INVALID


def test_bad_rows_written_inputs():
    kv = batch()
    bufs = {n: Fake(1 << 20) for n in ("pos", "seq", "inv_freq", "q_norm_w", "k_norm_w")}
    for n, b in bufs.items():
        assert rows_check(kv, qkv(**{n: b})) == OK and rows_check(kv, qkv(**{n: b, "q_out": b})) == INVALID
    cache, tables = Fake(1 << 20), Fake(1 << 20)
    assert rows_check(batch(k_cache=cache, v_cache=cache), qkv()) == INVALID
    for n in ("q", "k", "v", "q_out", "pos"):
        assert rows_check(batch(k_cache=cache), qkv(**{n: cache})) == INVALID
        assert rows_check(batch(v_cache=cache), qkv(**{n: cache})) == INVALID
    assert rows_check(batch(tables=tables), qkv(q_out=tables)) == INVALID


def decode(nh=6, **over):
    f = dict(q=Fake(4 * SEQS * nh * HD), out=Fake(4 * SEQS * nh * HD), seq_lens=Fake(4 * SEQS), ws=Fake(1 << 24),
             n_heads=nh, prefix_len=40, max_len=128)
    f.update(over)
    return DecodeRows(**f)


def decode_check(kv, r):
    return check("zh_check_decode_rows", kv.ptr, r.ptr, C.c_uint32(256))


def test_decode_accepted():
    for r in (decode(), decode(prefix_len=0), decode(prefix_len=128), decode(type=F16), decode(nh=32),
              decode(max_len=100, prefix_len=0, ws=None)):
        assert decode_check(batch(), r) == OK
    q = Fake(4 * SEQS * 6 * HD)
    assert decode_check(batch(), decode(q=q, out=q)) == OK


@pytest.mark.parametrize("over", [
    dict(n_heads=0), dict(n_heads=5), dict(n_heads=34), dict(max_len=0), dict(prefix_len=129), dict(q_off=16),
    dict(q_off=4), dict(q_stride=6 * HD - 4), dict(out_stride=6 * HD + 2), dict(seq_lens=Fake(16)), dict(out=None),
    dict(q=None)], ids=str)
def test_bad_decode(over):
    assert decode_check(batch(), decode(**over)) == INVALID


def test_bad_decode_workspace():
    """Refused where the call works in parts; a call of one part needs none."""
    kv = batch(table_stride=1024, tables=Fake(4 * SEQS * 1024))
    for ws in (None, Fake(64)):
        assert decode_check(kv, decode(max_len=16000, ws=ws)) == INVALID
        assert decode_check(kv, decode(max_len=16000, prefix_len=0, ws=ws)) == INVALID


def test_bad_decode_rest():
    assert decode_check(batch(), decode(max_len=129)) == TOO_LONG
    assert decode_check(batch(), decode(type=8)) == UNSUPPORTED
    assert decode_check(batch(head_dim=96), decode()) == INVALID
    wide = dict(table_stride=1 << 27, tables=Fake(4 * SEQS << 27))
    assert decode_check(batch(**wide), decode(max_len=(1 << 30) + 1, ws=Fake(1 << 40))) == INVALID
    one = Fake(1 << 30)
    for n in ("k_cache", "v_cache", "tables"):
        assert decode_check(batch(**{n: one}), decode(out=one)) == INVALID
        kv = dict(table_stride=1024, tables=Fake(4 * SEQS * 1024))
        kv[n] = one
        assert decode_check(batch(**kv), decode(max_len=16000, ws=Fake(1 << 30))) == OK
        assert decode_check(batch(**kv), decode(max_len=16000, ws=one)) == INVALID
    for n in ("q", "out", "seq_lens"):
        kv = batch(table_stride=1024, tables=Fake(4 * SEQS * 1024))
        assert decode_check(kv, decode(max_len=16000, ws=one, **{n: one})) == INVALID
    assert decode_check(batch(), decode(seq_lens=one, out=one)) == INVALID
    q = Fake(4 * SEQS * 8 * HD)
    assert decode_check(batch(), decode(q=q, out=q, out_off=4 * HD)) == INVALID


def test_decode_of_more_workgroups_than_a_launch_has():
    n = 1 << 22  # 2^23 workgroups: a launch of 2^31 threads and more
    kv = batch(n_seq=n, table_stride=1, tables=Fake(4 * n))
    big = dict(q=Fake(1 << 40), out=Fake(1 << 40), seq_lens=Fake(4 * n), ws=Fake(1 << 45), max_len=16)
    assert decode_check(kv, decode(prefix_len=0, **big)) == INVALID
    kv = batch(n_seq=n - 1, table_stride=1, tables=Fake(4 * n))
    assert decode_check(kv, decode(prefix_len=0, **big)) == OK


@pytest.mark.parametrize("n_seq,prefix", [(1, 0), (3, 300), (16, 0), (16, 4096), (40, 700), (64, 9000), (200, 8192)])
def test_workspace_for_a_length_serves_the_shorter_ones(n_seq, prefix):
    """A workspace is made for the largest max_len of a serving loop."""
    kv = batch(n_seq=n_seq, table_stride=4096, tables=Fake(4 * n_seq * 4096))
    q, out, lens = Fake(1 << 30), Fake(1 << 30), Fake(4 * n_seq)

    def need(max_len, t):
        lo, hi = 0, 1 << 40
        while lo < hi:
            mid = (lo + hi) // 2
            r = decode(q=q, out=out, seq_lens=lens, ws=Fake(mid), prefix_len=prefix, max_len=max_len, type=t)
            lo, hi = (lo, mid) if decode_check(kv, r) == OK else (mid + 1, hi)
        return lo

    for t in (0, F16):
        sizes = [need(max(prefix, 1) + own, t) for own in (0, 1, 16, 100, 130, 300, 500, 513, 700, 1100, 2000, 5000, 30000)]
        assert sizes == sorted(sizes)


def test_page_numbers_are_integers_of_32_bits():
    for bad in ([-1], [1 << 32], np.array([-1]), np.array([1 << 32]), np.array([1.5]), [[1]], ["a"]):
        with pytest.raises((ValueError, OverflowError, TypeError)):
            zinc_amd.hip._u32_array(bad)
    for good in ([7], np.array([7]), np.array([3, 7], dtype=np.uint32)[1:], np.arange(9, dtype=np.uint32)[7::9],
                 np.array([7], dtype=np.uint8)):
        p, n = zinc_amd.hip._u32_array(good)
        assert n == 1 and p._obj.value == 7
    assert zinc_amd.hip._u32_array([])[1] == 0 and zinc_amd.hip._u32_array(np.zeros(0, np.uint32))[1] == 0


def test_entries_refuse_a_null_context():
    L = zinc_amd.lib()
    assert L.zh_qk_norm_rope_kv_write_batched(None, batch().ptr, qkv().ptr) == INVALID
    assert L.zh_flash_decode_shared(None, batch().ptr, decode().ptr) == INVALID
    a = KvCaches([Fake(4096)], 16, 1, 64)
    p = np.zeros(1, dtype=np.uint32)
    assert L.zh_kv_copy_pages(None, a.ptr, a.ptr, p.ctypes.data, p.ctypes.data, 0) == INVALID
    assert L.zh_flash_decode_shared_ws(None, batch().ptr, 6, 0, 16) == 0
    assert L.zh_engine_fork_kv(None, None, 1) == INVALID

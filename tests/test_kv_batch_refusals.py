"""More of what the batched cache operators refuse, host side (no GPU)."""
import ctypes as C
import gc
import types

import pytest
from test_kv_batch import HD, INVALID, OK, Fake, batch, check, copy_check, decode, decode_check, qkv, rows_check

import zinc_amd
from zinc_amd import KvCaches, hip


def test_tables_whose_bytes_pass_64_bits():
    """4 * n_seq * table_stride is 2^64, which 64 bits hold as zero."""
    huge = dict(n_seq=1 << 31, table_stride=1 << 31)
    rows = qkv(n=4, seq=Fake(16))
    assert rows_check(batch(tables=Fake(1 << 20), **huge), rows) == INVALID
    assert check("zh_check_decode_rows", batch(tables=Fake(1 << 20), **huge).ptr, decode().ptr, C.c_uint32(256)) == INVALID
    # (2^32 - 1)^2 * 4 is 2^66 - 2^35 + 4, in 64 bits 2^64 - 2^35 + 4
    most = dict(n_seq=(1 << 32) - 1, table_stride=(1 << 32) - 1)
    assert rows_check(batch(tables=Fake(1 << 62), **most), rows) == INVALID


def test_rows_whose_bytes_pass_64_bits():
    """2^31 strides of 2^31 f32 elements are 2^64 bytes."""
    n, wide = (1 << 31) + 1, 1 << 31
    lists = dict(n_rows=n, pos=Fake(4 * n), seq=Fake(4 * n))
    ample = {k: Fake(4 * n * 6 * HD) for k in ("q", "k", "v", "q_out")}
    kv = batch()
    assert rows_check(kv, qkv(**lists, **ample)) == OK
    for name in ample:
        assert rows_check(kv, qkv(**lists, **ample, **{name + "_stride": wide})) == INVALID


class Owned(Fake):
    """A Fake whose free() is Buffer's (the library's own free left out)."""
    ctx = types.SimpleNamespace(h=None)
    free = hip.Buffer.free


@pytest.fixture()
def no_device_free(monkeypatch):
    monkeypatch.setattr(zinc_amd.lib(), "zh_buf_free", lambda ctx, buf: None)


def owned(plan, **sizes):
    bufs = {n: Owned(s) for n, s in sizes.items()}
    return plan(**bufs), bufs


@pytest.mark.parametrize("name", ["k_cache", "v_cache", "tables"])
def test_a_batch_of_a_freed_buffer(no_device_free, name):
    kv, bufs = owned(batch, **{n: 1 << 20 for n in ("k_cache", "v_cache", "tables")})
    assert rows_check(kv, qkv()) == OK and decode_check(kv, decode()) == OK
    bufs[name].free()
    assert rows_check(kv, qkv()) == INVALID and decode_check(kv, decode()) == INVALID
    assert zinc_amd.lib().zh_flash_decode_shared_ws(None, kv.ptr, 6, 0, 16) == 0


@pytest.mark.parametrize("name", ["q", "k", "v", "q_out", "pos", "seq", "inv_freq", "q_norm_w", "k_norm_w"])
def test_rows_of_a_freed_buffer(no_device_free, name):
    rows, bufs = owned(qkv, **{n: 1 << 20 for n in ("q", "k", "v", "q_out", "pos", "seq", "inv_freq", "q_norm_w", "k_norm_w")})
    assert rows_check(batch(), rows) == OK
    bufs[name].free()
    assert rows_check(batch(), rows) == INVALID


@pytest.mark.parametrize("name", ["q", "out", "seq_lens", "ws"])
def test_decode_rows_of_a_freed_buffer(no_device_free, name):
    rows, bufs = owned(decode, **{n: 1 << 24 for n in ("q", "out", "seq_lens", "ws")})
    assert decode_check(batch(), rows) == OK
    bufs[name].free()
    assert decode_check(batch(), rows) == INVALID


def test_caches_one_of_which_is_freed(no_device_free):
    bufs = [Owned(1 << 20) for _ in range(3)]
    a, b = (KvCaches(bufs, 64, 1, 64) for _ in range(2))
    assert copy_check(a, b, [1], [2]) == OK
    del b  # (a plan that is gone)
    bufs[1].free()
    assert copy_check(a, a, [1], [2]) == INVALID
    bufs[1].free()


def test_plans_leave_nothing_behind_in_their_buffers():
    """A loop that makes its plans anew, over caches that live on."""
    cache = Owned(1 << 20)
    for _ in range(100):
        batch(k_cache=cache)
    gc.collect()
    assert len(cache._plans) == 0

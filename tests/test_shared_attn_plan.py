"""How zh_flash_decode_shared cuts a call and what workspace it asks for, host
side (no GPU)."""
import ctypes as C

import numpy as np
import pytest
from test_kv_batch import Fake, OK, batch, decode, decode_check

import zinc_amd
from zinc_amd import F16, F32

K, V, TABLES = (Fake(1 << 45) for _ in range(3))


def batch_of(n_seq, nkv, hd):
    return batch(k_cache=K, v_cache=V, tables=TABLES, n_seq=n_seq, table_stride=1 << 16,
                 n_kv_heads=nkv, head_dim=hd)


def plan(n_seq, nh, nkv, hd, prefix, max_len, t, cus=256):
    """(tile, parts of the prefix, own parts, bytes of ws)"""
    out = (C.c_uint64 * 4)()
    f = zinc_amd.lib().zh_check_shared_plan
    assert f(batch_of(n_seq, nkv, hd).ptr, C.c_uint32(nh), C.c_uint32(prefix), C.c_uint32(max_len), C.c_uint32(t),
             C.c_uint32(cus), out) == OK
    return tuple(out)


def workspace(n_seq, nh, nkv, hd, prefix, max_len, cus=256):
    f = zinc_amd.lib().zh_check_shared_ws
    f.restype = C.c_uint64
    return f(batch_of(n_seq, nkv, hd).ptr, C.c_uint32(nh), C.c_uint32(prefix), C.c_uint32(max_len), C.c_uint32(cus))


@pytest.mark.parametrize("full,smaller", [
    ((256, 32, 8, 128, 0, 512), (170, 0, 512)),        # sequences end
    ((256, 32, 8, 128, 0, 512), (64, 0, 512)),
    ((256, 32, 8, 128, 1, 4608), (256, 0, 4608)),      # a prefix goes
    ((64, 32, 8, 128, 16384, 16900), (48, 9000, 9400)),  # it gets shorter, and its tiles fewer
    ((64, 64, 4, 64, 4000, 4100), (1, 4000, 4100)),
    ((130, 32, 8, 128, 8192, 8300), (129, 8192, 8300)),
    ((200, 2, 1, 128, 30000, 34000), (3, 30000, 31000))], ids=str)
def test_workspace_of_a_full_batch_serves_its_remains(full, smaller):
    n, prefix, max_len = smaller
    for t in (F32, F16):
        assert plan(n, *full[1:4], prefix, max_len, t)[3] <= workspace(*full)


def test_workspace_serves_every_smaller_call():
    """Any n_seq, prefix and max_len up to those it was asked for, on devices of
    several sizes."""
    rng = np.random.default_rng(17)

    def log_int(lo, hi):
        return int(np.exp(rng.uniform(np.log(lo), np.log(hi + 1))))

    for _ in range(4000):
        nkv, G, hd, cus = log_int(1, 64), int(rng.integers(1, 17)), int(rng.choice([64, 128])), int(rng.choice([64, 256, 304]))
        n, prefix, own = log_int(1, 2000), int(rng.integers(4) > 0) * log_int(1, 200000), log_int(1, 20000)
        ws = workspace(n, nkv * G, nkv, hd, prefix, prefix + own, cus)
        for _ in range(4):
            m, p = log_int(1, n), int(rng.integers(2)) * (log_int(1, prefix) if prefix else 0) or prefix
            length = int(rng.integers(max(p, 1), prefix + own + 1))
            for t in (F32, F16):
                assert plan(m, nkv * G, nkv, hd, p, length, t, cus)[3] <= ws


def test_the_check_asks_for_the_plan_s_bytes():
    n, nh, nkv, hd, prefix, max_len = 40, 32, 8, 128, 700, 1500
    need = plan(n, nh, nkv, hd, prefix, max_len, F32)[3]
    row = Fake(1 << 30), Fake(1 << 30), Fake(4 * n)
    for size, ok in ((need, True), (need - 1, False)):
        r = decode(nh=nh, q=row[0], out=row[1], seq_lens=row[2], ws=Fake(size), prefix_len=prefix, max_len=max_len)
        assert (decode_check(batch_of(n, nkv, hd), r) == OK) is ok


def test_workspace_of_refused_sizes():
    assert workspace(4, 6, 4, 128, 0, 16) == 0 and workspace(4, 8, 4, 96, 0, 16) == 0
    assert workspace(4, 8, 4, 128, 17, 16) == 0 and workspace(1 << 23, 1, 1, 128, 0, 16) == 0

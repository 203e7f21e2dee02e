"""More of what the batched cache operators refuse, host side (no GPU)."""
import ctypes as C

from test_kv_batch import HD, INVALID, OK, Fake, batch, check, decode, qkv, rows_check


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

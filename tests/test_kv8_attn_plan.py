"""How attention over the 8-bit cache deals its streamed rows out, host side (no GPU): a
call whose workgroups each take a whole sequence needs no workspace."""
import pytest
from test_kv8_refusals import AttnRows, Fake, Kv8Batch, attn_check
from test_kv_batch import INVALID, OK

from zinc_amd import E4M3, F16


def whole(n_seq, max_len, nkv, hd, G, rows=1):
    kv = Kv8Batch(*[Fake(1 << 32) for _ in range(6)], row_start=Fake(1 << 32), n_seq=n_seq, table_stride=max_len // 16 + 1,
                  cache_tokens=16, n_kv_heads=nkv, head_dim=hd, type=E4M3)
    kv_rows = dict(q=Fake(1 << 40), out=Fake(1 << 40), n_rows=n_seq * rows, max_rows=rows, max_len=max_len, n_heads=G * nkv, type=F16)
    rc = attn_check(kv, AttnRows(ws=None, **kv_rows))
    assert attn_check(kv, AttnRows(ws=Fake(1 << 36), **kv_rows)) == OK and rc in (OK, INVALID)
    return rc == OK


@pytest.mark.parametrize("nkv,hd,rows,n_seq,up_to,from_", [
    (8, 128, 1, 16, 1000, 1600), (8, 128, 1, 200, 4000, 6000), (8, 128, 1, 800, 12000, 27000),
    (8, 128, 1, 1600, 35000, 52000), (8, 64, 1, 64, 1700, 3000), (8, 64, 1, 600, 9000, 18000), (8, 64, 1, 800, 11000, 23000),
    (8, 64, 1, 1600, 22000, 46000), (4, 64, 5, 200, 3000, 4800), (4, 64, 5, 400, 5000, 8900), (8, 128, 5, 16, 1000, 2000),
    (1, 128, 1, 6400, 60000, 120000), (8, 128, 1, 200000, 100, 1 << 31)])
def test_a_whole_sequence_a_workgroup(nkv, hd, rows, n_seq, up_to, from_):
    """Up to lengths that a batch can have in one sequence alone: one long sequence among
    many short ones is not left to one workgroup however many the others are."""
    assert whole(n_seq, up_to, nkv, hd, 4, rows)
    assert from_ > 1 << 30 or not whole(n_seq, from_, nkv, hd, 4, rows)


def test_so_many_that_the_join_would_not_fit_a_launch():
    assert whole(1 << 18, 1 << 13, 4, 64, 1) and not whole((1 << 10) - 1, 1 << 20, 4, 64, 1)

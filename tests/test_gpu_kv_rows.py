"""q/k norm + rotation + KV write of many rows (zh_qk_norm_rope_kv_write_batched):
calls that name a slot more than once."""
import numpy as np
import pytest
from test_gpu_kv_batch import ctx, zh  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [128, 96])  # (96: the kernel of any shape)
def test_rows_that_name_the_same_slot(zh, ctx, hd):  # noqa: F811
    """600 rows of a sequence, 200 positions three times each: every element of a
    slot is one of its three rows', no other slot is written, every q is its row's."""
    rng = np.random.default_rng(41)
    T, nq, nkv, tokens = 600, 4, 2, 256
    x = rng.standard_normal((T, nq + 2 * nkv, hd)).astype(np.float16)
    pos = np.arange(T) % 200
    kc0 = rng.standard_normal((nkv, tokens, hd)).astype(np.float16)
    pages = rng.permutation(tokens // 16).astype(np.uint32)
    u = ctx.upload
    X, K, V, out = u(x), u(kc0), u(kc0), ctx.alloc(2 * T * nq * hd)
    kv = zh.KvBatch(K, V, u(pages), 1, pages.size, tokens, nkv, hd)
    w = (nq + 2 * nkv) * hd
    rows = zh.QkvRows(q=X, k=X, v=X, k_off=2 * nq * hd, v_off=2 * (nq + nkv) * hd, q_stride=w, k_stride=w, v_stride=w,
                      q_out=out, type=zh.F16, pos=u(pos.astype(np.uint32)), seq=u(np.zeros(T, np.uint32)), n_rows=T,
                      n_q_heads=nq)  # (no norm, no rotation: the rows as they are)
    ctx.qk_norm_rope_kv_write_batched(kv, rows)
    ctx.sync()
    assert np.array_equal(out.download(np.float16, T * nq * hd).reshape(T, nq, hd), x[:, :nq])
    slot = pages[np.arange(200) // 16].astype(np.int64) * 16 + np.arange(200) % 16
    for buf, first in ((K, nq), (V, nq + nkv)):
        got = buf.download(np.float16, kc0.size).reshape(kc0.shape)
        written = got[:, slot].transpose(1, 0, 2)  # [position][head][dim]
        theirs = x[:, first:first + nkv].reshape(3, 200, nkv, hd)
        assert (written[None] == theirs).any(0).all()
        rest = np.ones(tokens, bool)
        rest[slot] = False
        assert np.array_equal(got[:, rest], kc0[:, rest])

"""The batched cache operators over caches of 8 GiB each: rows written to pages at
their ends, attended there in both forms, copied to the low pages and attended again."""
import numpy as np
import pytest
from test_gpu_kv_batch import NP_TYPE, attend64, close, ctx, zh  # noqa: F401
from test_shared_attn_plan import plan

pytestmark = pytest.mark.gpu


def test_caches_past_32_bits(zh, ctx):  # noqa: F811
    rng = np.random.default_rng(61)
    nkv, G, hd, tokens, S, P = 2, 16, 128, 1 << 24, 62, 2827
    lens = [P + 1 + i % 3 for i in range(S)]
    nh, full, stride, last = nkv * G, P // 16, P // 16 + 1, tokens // 16
    own = full + np.arange(S)  # (each its own page past the full ones: the prefix's last 11 tokens and its own)
    near = np.concatenate([np.tile(np.arange(full), (S, 1)), own[:, None]], 1).astype(np.uint32)
    far = (last - 1 - near).astype(np.uint32)
    # K and V of the near pages on the host: the prefix's tokens alike in every own page
    shape = (nkv, (full + S) * 16, hd)
    kc, vc = (rng.standard_normal(shape, dtype=np.float32).astype(np.float16) for _ in range(2))
    for c in (kc, vc):
        p = c.reshape(nkv, -1, 16, hd)
        p[:, full:, :P % 16] = p[:, full:full + 1, :P % 16]
    # one row a token: the full pages' through sequence 0, then each own page's
    pos = np.concatenate([np.arange(full * 16)] + [np.arange(full * 16, n) for n in lens])
    seq = np.concatenate([np.zeros(full * 16, int)] + [np.full(n - full * 16, s) for s, n in enumerate(lens)])
    at = near[seq, pos // 16].astype(np.int64) * 16 + pos % 16
    x = np.concatenate([rng.standard_normal((len(pos), nh, hd)).astype(np.float16), kc[:, at].transpose(1, 0, 2),
                        vc[:, at].transpose(1, 0, 2)], 1)
    u = ctx.upload
    K, V = (ctx.alloc(2 * nkv * tokens * hd) for _ in range(2))
    X, TN, TF, L = u(x), u(near), u(far), u(np.array(lens, np.uint32))
    far_kv, near_kv = (zh.KvBatch(K, V, t, S, stride, tokens, nkv, hd) for t in (TF, TN))
    w = (nh + 2 * nkv) * hd
    ctx.qk_norm_rope_kv_write_batched(far_kv, zh.QkvRows(
        q=X, k=X, v=X, k_off=2 * nh * hd, v_off=2 * (nh + nkv) * hd, q_stride=w, k_stride=w, v_stride=w, type=zh.F16,
        q_out=ctx.alloc(2 * len(pos) * nh * hd), pos=u(pos.astype(np.uint32)), seq=u(seq.astype(np.uint32)),
        n_rows=len(pos), n_q_heads=nh))
    ctx.sync()
    q = rng.standard_normal((S, nh, hd))
    got = {}
    for kv, name in ((far_kv, "far"), (near_kv, "near")):
        if name == "near":
            pages = np.unique(near)
            s = zh.KvCaches([K, V], tokens, nkv, hd)
            ctx.kv_copy_pages(s, s, pages, last - 1 - pages)
        for t, tile in ((zh.F32, 0), (zh.F16, 2)):
            assert plan(S, nh, nkv, hd, P, P + 3, t, ctx.info()[1])[0] == tile
            Q, out = u(q.astype(NP_TYPE[t])), ctx.alloc(S * nh * hd * 4)
            ctx.flash_decode_shared(kv, zh.DecodeRows(
                q=Q, out=out, seq_lens=L, ws=ctx.alloc(ctx.flash_decode_shared_ws(kv, nh, P, P + 3)), n_heads=nh,
                prefix_len=P, max_len=P + 3, type=t))
            ctx.sync()
            got[name, t] = out.download(NP_TYPE[t], S * nh * hd).reshape(S, nh, hd)
    for t in (zh.F32, zh.F16):
        assert np.array_equal(got["far", t], got["near", t])
        only = [0, 7, 30, S - 1]
        want, tol = attend64(q.astype(NP_TYPE[t]), kc, vc, near, lens, hd ** -0.5, t, P, only)
        close(got["far", t].astype(np.float64)[only], want[only], tol[only])

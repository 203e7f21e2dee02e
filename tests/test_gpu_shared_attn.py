"""Decode attention with a shared prefix (zh_flash_decode_shared): queries and
scales of any size, against the module's formula in 64 bits (the bounds are
test_gpu_kv_batch's, the same for both forms of the prefix)."""
import numpy as np
import pytest
from test_gpu_kv_batch import NP_TYPE, attend64, close, ctx, make, run_attention, store_error, zh  # noqa: F401

pytestmark = pytest.mark.gpu

# q heads, kv heads, head_dim, prefix, lengths: streamed, and through LDS tiles (f32 too)
STREAMED = (8, 2, 128, 100, [140, 139])
TILES = (64, 4, 64, 2301, [2302 + 7 * i % 90 for i in range(62)])
FORMS = pytest.mark.parametrize("case", [STREAMED, TILES], ids=["streamed", "tiles"])


def inputs(case, seed):
    nh, nkv, hd, P, lens = case
    rng = np.random.default_rng(seed)
    kc, vc, tables, _, M = make(rng, len(lens), nkv, hd, P, lens)
    return rng.standard_normal((len(lens), nh, hd)), kc, vc, tables, lens, P, M


def checked(lens):
    """Every 7th sequence and the last (of tiles: rows of every wave)."""
    return sorted({*range(0, len(lens), 7), len(lens) - 1})


@FORMS
@pytest.mark.parametrize("size", [-128, -124, 119, 125])
def test_f32_queries_of_the_type_s_whole_range(zh, ctx, case, size):  # noqa: F811
    """Queries of 2^size, subnormal ones and ones up to the type's largest among
    them, whose scores the scale brings back to ordinary ones."""
    q, kc, vc, tables, lens, P, M = inputs(case, 300 + size)
    with np.errstate(under="ignore"):
        q = (q * 2.0 ** size).astype(np.float32)
    scale = float(np.float32(min(0.09 * 2.0 ** -size, 3e38)))
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 0, scale=scale)
    only = checked(lens)
    want, tol = attend64(q, kc, vc, tables, lens, scale, 0, P, only)
    close(got[only], want[only], tol[only])


@FORMS
def test_f32_queries_with_one_large_dim(zh, ctx, case):  # noqa: F811
    """A dim of the queries 2^16 times the others, where K is zero: the scores are the
    others' (q's smaller dims keep 2^-39 of the largest: here 2^-23 of a typical one)."""
    q, kc, vc, tables, lens, P, M = inputs(case, 9)
    q[:, :, 5] = 2.0 ** 16 * np.where(np.arange(case[0]) % 2, 1, -1)
    kc[:, :, 5] = 0
    q = q.astype(np.float32)
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 0)
    only = checked(lens)
    want, tol = attend64(q, kc, vc, tables, lens, case[2] ** -0.5, 0, P, only)
    close(got[only], want[only], tol[only])


@FORMS
@pytest.mark.parametrize("t,size,scale", [(0, 1e-30, 1e-30), (0, 1e-38, -1e-38), (0, 1.0, 1e-44), (1, 1.0, -1e-44)])
def test_scores_too_small_to_tell_tokens_apart(zh, ctx, case, t, size, scale):  # noqa: F811
    """Scores below 2^-60: every weight alike, nothing masked among them (scale *
    log2 e times a query's power of two is no f32 any more)."""
    q, kc, vc, tables, lens, P, M = inputs(case, 7)
    q = (q * size).astype(NP_TYPE[t])
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, scale=scale)
    only = checked(lens)
    want, tol = attend64(q, kc, vc, tables, lens, scale, t, P, only)
    close(got[only], want[only], tol[only])


@FORMS
@pytest.mark.parametrize("t,size,scale", [(0, 1e30, 1e30), (0, 1e37, -3e38), (1, 1.0, 3e38)])
def test_scores_too_large_for_f32(zh, ctx, case, t, size, scale):  # noqa: F811
    """The token of the largest score has all of the weight, where it stands out by
    more than the products' error (2^-18 of the sum of their magnitudes)."""
    q, kc, vc, tables, lens, P, M = inputs(case, 8)
    q = (q * size).astype(NP_TYPE[t])
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, scale=scale)
    G, rows = case[0] // case[1], 0
    for s in checked(lens):
        tk = np.arange(lens[s])
        at = tables[np.where(tk < P, 0, s), tk // 16].astype(np.int64) * 16 + tk % 16
        for h in range(case[0]):
            k = kc[h // G, at].astype(np.float64)
            x = q[s, h].astype(np.float64) / size
            sc = np.sign(scale) * (k @ x)
            a, b = np.sort(sc)[-2:]
            if b - a > 2.0 ** -15 * (np.abs(k) @ np.abs(x)).max():
                want = vc[h // G, at[sc.argmax()]].astype(np.float64)
                assert (np.abs(got[s, h] - want) <= np.abs(want) * 2.0 ** -20 + store_error(t, want)).all(), (s, h)
                rows += 1
    assert rows > len(checked(lens)) * case[0] // 2

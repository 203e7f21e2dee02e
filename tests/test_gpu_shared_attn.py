"""Decode attention with a shared prefix (zh_flash_decode_shared): queries and
scales of any size, the form that a case is meant for, f16 results rounded once,
against the formula in 64 bits (the bounds are test_gpu_kv_batch's, the same for
both forms of the prefix)."""
import numpy as np
import pytest
from test_gpu_kv_batch import NP_TYPE, attend64, close, ctx, make, run_attention, store_error, zh  # noqa: F401

from test_shared_attn_plan import plan

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


# Through LDS tiles in both types: q heads, kv heads, head_dim, prefix, lengths, scale, rows of a
# workgroup / 128. The prefixes end 1 to 61 tokens into a stage of 64.
TILED = [
    (128, 8, 128, 1527, [0, 1527, 5] + [1528 + 3 * i % 31 for i in range(59)], 0.09, 2),  # 992 rows
    (128, 8, 64, 1153, [1153, 3] + [1154 + i % 19 for i in range(60)], -0.11, 2),
    (512, 32, 128, 3361, [3361 + 17 * i for i in range(7)], -0.09, 1),                   # 112 rows
    (512, 32, 64, 2506, [2507, 40, 2506, 2600, 2510, 2511, 2512], 0.125, 1),
    (128, 8, 128, 1527, [1528 + 19 * i % 1100 for i in range(62)], 0.09, 2),             # own tokens in parts
    (24, 8, 128, 5221, [5222 + i % 40 for i in range(91)], 0.09, 2),                     # 273 rows, 3 a sequence
]


def relative_rms(got, want):
    return np.sqrt(np.square(got - want).sum() / np.square(want).sum())


# Beside the bound of every element, one of their root mean square: rounding errors of many tokens
# and dims are as often up as down. f32: a score of up to 8 within 2^-22 of itself moves a weight by
# 2^-19, the weights' two pieces and exp2 by 2^-21, some hundred sums by 10 2^-24: below 2^-18, and
# the limit is 2^-17. One fp16 piece of q or of the weights alone is 2^-13 (test_shared_attn_bound).
# f16: the weights' one piece and the store's rounding, 2^-11 / 12^(1/2) of a value on its average
# octave each: below 2^-11.
RMS = {0: 2.0 ** -17, 1: 2.0 ** -11}


@pytest.mark.parametrize("t", [0, 1], ids=["f32", "f16"])
@pytest.mark.parametrize("case", TILED + [(*STREAMED, 0.09, 0)],
                         ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
def test_attention_in_the_form_it_is_meant_for(zh, ctx, case, t):  # noqa: F811
    """Rows of every wave (32 rows) of a workgroup."""
    nh, nkv, hd, P, lens, scale, tile = case
    q, kc, vc, tables, _, _, M = inputs(case[:5], nh + P)
    q = (q * 1.5).astype(NP_TYPE[t])
    way = plan(len(lens), nh, nkv, hd, P, M, t, ctx.info()[1])
    assert way[0] == tile and (tile == 0 or way[2] == (3 if max(lens) > P + 1000 else 1))
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, t, scale=scale)
    G = nh // nkv
    only = [s for s in range(len(lens)) if s == 0 or s * G // 32 != (s - 1) * G // 32 or s == len(lens) - 1]
    want, tol = attend64(q, kc, vc, tables, lens, scale, t, P, only)
    close(got[only], want[only], tol[only])
    assert relative_rms(got[only], want[only]) < RMS[t]


@pytest.mark.parametrize("case", [STREAMED, (32, 8, 128, 300, [400, 500, 301, 7]), (16, 2, 64, 0, [900, 1, 33, 1300]),
                                  (64, 4, 128, 1237, [1238 + i for i in range(60)])],
                         ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}-{len(c[4])}x{max(c[4])}")
def test_f16_results_are_rounded_once_where_the_prefix_is_streamed(zh, ctx, case):  # noqa: F811
    """Against the formula's results rounded to fp16. What is within 2^-18 before that
    rounding is off by a step (2^-10 at most) in one of 2^8 at most: a root mean square
    below (2^-18 2^-10)^(1/2) = 2^-14. With weights of 11 bits most results are off by
    2^-13 before it: (2^-13 2^-10)^(1/2) = 2^-11.5. The limit is 2^-13."""
    nh, nkv, hd, P, lens = case
    q, kc, vc, tables, _, _, M = inputs(case, 51)
    q = (q * 1.5).astype(np.float16)
    assert plan(len(lens), nh, nkv, hd, P, M, 1, ctx.info()[1])[0] == 0
    got = run_attention(zh, ctx, q, kc, vc, tables, lens, P, M, 1)
    only = checked(lens)
    want, tol = attend64(q, kc, vc, tables, lens, hd ** -0.5, 1, P, only)
    close(got[only], want[only], tol[only])
    assert relative_rms(got[only], want[only].astype(np.float16).astype(np.float64)) < 2.0 ** -13

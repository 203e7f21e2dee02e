"""How exact the 8-bit cache's operators are, in every form that a call can take: f16
attention rounded once."""
import kv8_ref as ref
import numpy as np
import pytest
from test_gpu_kv8 import E4M3, I8, Cache, attend, close, ctx, expect, tables_for, tolerance, zh  # noqa: F401
from test_gpu_kv8_edges import starts_of
from test_gpu_shared_attn import relative_rms

pytestmark = pytest.mark.gpu

# counts, lens, heads per kv head, kv heads, head_dim. LDS tiles: more than 192 query rows of a
# sequence and kv head
FORMS = [
    ([1, 1, 1], [3000, 900, 2100], 4, 2, 128),                  # streamed, in shares
    ([20, 60], [60, 300], 3, 1, 64),                            # streamed, a sequence a workgroup
    ([260, 3], [700, 300], 1, 2, 64),                           # tiles whole, short rows among them
    ([300, 1, 1], [4000, 1000, 33], 1, 1, 128),                 # tiles cut, decode rows on tiles
    ([50], [2600], 4, 1, 128),
    ([150, 2, 2, 2, 2, 2, 2, 2, 2, 2], [900] + [500] * 9, 2, 1, 64),  # tiles beside streamed rows
]


@pytest.mark.parametrize("fmt", [I8, E4M3])
@pytest.mark.parametrize("case", FORMS, ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[2]}-{c[4]}")
def test_f16_attention_is_rounded_once(zh, ctx, fmt, case):  # noqa: F811
    """Against the formula's results rounded to fp16. What is within 2^-18 before that
    rounding is off by a step (2^-10 at most) in one of 2^8 at most: a root mean square
    below (2^-18 2^-10)^(1/2) = 2^-14. With weights of 11 bits most results are off by
    2^-13 before it: (2^-13 2^-10)^(1/2) = 2^-11.5 (test_kv8_pieces). The limit is 2^-13,
    for each sequence by itself, so that few rows beside many count."""
    counts, lens, G, nkv, hd = case
    rng = np.random.default_rng(sum(counts) + hd)
    tables, total = tables_for(rng, lens, 2)
    cache = Cache(ctx, rng, total, nkv, hd, fmt)
    starts = starts_of(counts)
    q, got = attend(zh, ctx, rng, cache, tables, counts, lens, G, 1, None if max(counts) == 1 else starts)
    want, *terms = expect(cache, tables, q, counts, lens, hd ** -0.5)
    close(got, want, tolerance(cache, 1, want, *terms, lens, floor=-29))
    for a, b in zip(starts[:-1], starts[1:]):
        assert relative_rms(got[a:b], want[a:b].astype(np.float16).astype(np.float64)) < 2.0 ** -13

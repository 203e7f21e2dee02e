"""The root mean square limit of the shared-prefix attention's f32 tests tells two
fp16 pieces from one (no GPU): the prefix's weights and products emulated with one
piece of q, of the weights or of both, and with two."""
import numpy as np
import pytest
from test_gpu_shared_attn import RMS, TILED, relative_rms


def pieces(x, n):
    """x as the sum of n fp16 values."""
    total = np.zeros_like(x)
    for _ in range(n):
        total += (x - total).astype(np.float16)
    return total


@pytest.mark.parametrize("np_q,np_p", [(2, 2), (1, 2), (2, 1), (1, 1)])
@pytest.mark.parametrize("case", TILED, ids=lambda c: f"{c[0]}-{c[1]}-{c[2]}-{c[3]}")
def test_limit_of_one_piece_and_two(case, np_q, np_p):
    P, hd, scale = case[3], case[2], case[5]
    rng = np.random.default_rng(P)
    k, v = (rng.standard_normal((P, hd)).astype(np.float16).astype(np.float64) for _ in range(2))
    q = (rng.standard_normal((64, hd)) * 1.5).astype(np.float32).astype(np.float64)

    def attention(x, n):
        s = x @ k.T * scale
        w = np.exp(s - s.max(1, keepdims=True))
        return (pieces(w * 256, n) if n else w * 256) @ v / (w.sum(1, keepdims=True) * 256)

    top = np.abs(q).max(1, keepdims=True)
    up = 2.0 ** (14 - np.floor(np.log2(top)))
    err = relative_rms(attention(pieces(q * up, np_q) / up, np_p), attention(q, 0))
    if np_q == np_p == 2:
        assert err < RMS[0] / 16
    else:
        assert err > 4 * RMS[0]

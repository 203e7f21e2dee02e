"""The root mean square limit of the 8-bit attention's f16 test tells weights in two
fp16 pieces from one (no GPU): the products emulated with either."""
import kv8_ref as ref
import numpy as np
import pytest


def pieces(x, n):
    """x as the sum of n fp16 values."""
    total = np.zeros_like(x)
    for _ in range(n):
        total += (x - total).astype(np.float16)
    return total


@pytest.mark.parametrize("fmt", [ref.I8, ref.E4M3])
@pytest.mark.parametrize("n,hd", [(300, 64), (1000, 128), (2600, 128), (4000, 64)])
def test_limit_of_one_piece_and_two(fmt, n, hd):
    rng = np.random.default_rng(n)
    codes = ref.encode(np.clip(rng.normal(size=(2, n, hd)) * (40 if fmt == ref.I8 else 100), *((-127, 127) if fmt == ref.I8 else (-448, 448))), fmt)
    k, v = ref.decode(codes, fmt) * 2.0 ** (-6 if fmt == ref.I8 else -7)
    q = (rng.normal(size=(64, hd)) * 2).astype(np.float16).astype(np.float64)
    s = q @ k.T * hd ** -0.5
    w = np.exp(s - s.max(1, keepdims=True))
    want = (w @ v / w.sum(1, keepdims=True)).astype(np.float16).astype(np.float64)

    def off(count):
        got = (pieces(w * 16, count) @ v / (w.sum(1, keepdims=True) * 16)).astype(np.float16).astype(np.float64)
        return np.sqrt(np.square(got - want).sum() / np.square(want).sum())

    assert off(2) < 2.0 ** -14 and off(1) > 2.0 ** -12.5

"""The plain form of the 8-bit cache that the other tests compare with, against
torch's e4m3 and what the formats' definitions fix."""
import kv8_ref as ref
import numpy as np
import pytest
import torch


def test_e4m3_numbers_and_rounding_are_torchs():
    v = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(v, ref.E4M3_VALUES, equal_nan=True)
    rng = np.random.default_rng(1)
    mid = np.unique(np.abs(v[np.isfinite(v)]))
    x = np.concatenate([mid, (mid[1:] + mid[:-1]) / 2, rng.normal(size=4000) * 100, rng.normal(size=1000) * 2.0 ** -8])
    x = np.clip(np.concatenate([x, -x]), -448, 448).astype(np.float32)
    got = ref.encode(x.astype(np.float64), ref.E4M3)
    assert np.array_equal(got, torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


@pytest.mark.parametrize("fmt", [ref.I8, ref.E4M3])
def test_least_scale(fmt):
    top = ref.LARGEST[fmt]
    assert ref.least_scale(0, fmt) == 2.0 ** -64 and ref.least_scale(top, fmt) == 1
    assert ref.least_scale(np.nextafter(top, 1e9), fmt) == 2 and ref.least_scale(top * 2.0 ** 64, fmt) == 2.0 ** 64
    assert np.isnan(ref.least_scale(top * 2.0 ** 64 * 1.01, fmt)) and np.isnan(ref.least_scale(np.inf, fmt))


@pytest.mark.parametrize("fmt", [ref.I8, ref.E4M3])
def test_error_after_any_number_of_rises(fmt):
    """Tokens of growing size, one at a time: i8 less than one step of the last
    scale off, e4m3 half a step of the value and one of the subnormals."""
    rng = np.random.default_rng(2)
    codes, scale = np.zeros((16, 64), dtype=np.uint8), np.nan
    x = rng.normal(size=(16, 64)) * 1.7 ** np.arange(16)[:, None]
    for i in range(16):
        codes, scale = ref.store_page(codes, scale, fmt, [i], x[i:i + 1])
    err = np.abs(ref.decode(codes, fmt) * scale - x)
    if fmt == ref.I8:
        assert (err < scale).all()
    else:
        # rounded once as a normal number; below 2^-6 each rise rounds to halves of 2^-9 again: less than 2^-9 in all
        assert (err <= np.abs(x) * 2.0 ** -4 + scale * 2.0 ** -9).all()

"""The 8-bit KV cache in plain numpy, in 64 bits: its two formats, the quantised
write of a batch's rows, and attention over it."""
import numpy as np

I8, E4M3 = 24, 256
LARGEST = {I8: 127.0, E4M3: 448.0}


def _e4m3_values():
    v = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = np.nan if c & 127 == 127 else -x if c & 128 else x
    return v


E4M3_VALUES = _e4m3_values()


def decode(codes, fmt):
    return codes.view(np.int8).astype(np.float64) if fmt == I8 else E4M3_VALUES[codes]


def encode(x, fmt):
    """Numbers within the format's largest to codes, to nearest, ties to even."""
    if fmt == I8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    e = np.where(a == 0, -6, np.maximum(np.frexp(a)[1] - 1, -6))  # the binade's exponent
    k = np.rint(a * 2.0 ** (3 - e)).astype(np.int64)  # 8 .. 16 (below 2^-6: 0 .. 8)
    code = k + 8 * (e + 6)  # the carry into the next binade falls out of the sum
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def least_scale(top, fmt):
    """2^e with the least e for which top <= largest * 2^e; NaN where that passes 2^64."""
    if not np.isfinite(top):
        return np.nan
    e = -64
    while top > LARGEST[fmt] * 2.0 ** e:
        e += 1
    return 2.0 ** e if e <= 64 else np.nan


def usable(s):
    return np.isfinite(s) and 2.0 ** -64 <= s <= 2.0 ** 64


def store_page(codes, scale, fmt, slots, rows):
    """rows [n][hd] into the slots of one block: codes u8 [16][hd], its scale. Returns both."""
    codes = codes.copy()
    need = least_scale(np.abs(rows).max() if np.isfinite(rows).all() else np.inf, fmt)
    begun = 0 in slots
    new = need if begun else max(need, scale) if usable(scale) and need == need else np.nan
    if begun:
        codes[[i for i in range(16) if i not in slots]] = 0
    elif new == new and new != scale:
        codes = encode(decode(codes, fmt) * (scale / new), fmt)
    codes[slots] = encode(rows / new, fmt) if new == new else 0
    return codes, new


def turned(x, w, freq, pos, eps, rd):
    """x [n][heads][hd] normalised and rotated."""
    x = x.astype(np.float64)
    if w is not None:
        x = w.astype(np.float64) * (x * (1 / np.sqrt((x * x).sum(-1, keepdims=True) / x.shape[-1] + np.float64(np.float32(eps)))))
    y, h = x.copy(), rd // 2
    if h:
        th = (pos.astype(np.float64)[:, None] * freq.astype(np.float64))[:, None]
        a, b = x[..., :h], x[..., h:rd]
        y[..., :h], y[..., h:rd] = a * np.cos(th) - b * np.sin(th), a * np.sin(th) + b * np.cos(th)
    return y


def attention(q, kc, vc, ks, vs, table, n_own, length, scale, fmt):
    """q [n][nh][hd]: the last n_own of `length` tokens. Returns out, for each output
    the sum of w |v| and what a weight off by the row's largest one w b would make,
    (sum of |Vc|) max(w b), and for each row and head the largest sum of |q k| scale."""
    n, nh, hd = q.shape
    nkv = kc.shape[0]
    t = np.arange(length)
    at = table[t // 16].astype(np.int64) * 16 + t % 16
    out, mag, unit, big = *(np.zeros((n, nh, hd)) for _ in range(3)), np.zeros((n, nh))
    for h in range(nkv):
        k = decode(kc[h, at], fmt) * ks[at // 16, h][:, None].astype(np.float64)
        vcodes, b = np.abs(decode(vc[h, at], fmt)), vs[at // 16, h].astype(np.float64)
        v = decode(vc[h, at], fmt) * b[:, None]
        for g in range(h * nh // nkv, (h + 1) * nh // nkv):
            for i in range(n):
                m = length - n_own + i + 1
                if m <= 0:
                    continue
                s = scale * (k[:m] @ q[i, g].astype(np.float64))
                w = np.exp(s - s.max())
                w /= w.sum()
                out[i, g], mag[i, g] = w @ v[:m], w @ np.abs(v[:m])
                unit[i, g] = vcodes[:m].sum(0) * (w * b[:m]).max()
                big[i, g] = abs(scale) * (np.abs(k[:m]) @ np.abs(q[i, g].astype(np.float64))).max()
    return out, mag, unit, big

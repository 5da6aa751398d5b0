"""Rows in 8 bits and group norm in 64 bits, from their definitions (numpy on
the CPU), for the tests of ien_quantize8, ien_multiply8 and ien_group_norm."""

import numpy as np

# Every e4m3 value by its byte: sign, 4 exponent bits (bias 7), 3 of mantissa;
# 0x7f and 0xff are NaN.
_MAGNITUDES = np.array([(b & 7) * 2.0**-9 if b < 8 else (8 + (b & 7)) * 2.0 ** ((b >> 3) - 10) for b in range(127)])
E4M3 = np.concatenate([_MAGNITUDES, [np.nan], -_MAGNITUDES, [np.nan]])


def to_bytes(v):
    """f64 values of at most 448 as e4m3 bytes, to nearest, ties to even."""
    m = np.abs(v)
    low = np.clip(np.searchsorted(_MAGNITUDES, m, side="right") - 1, 0, 126)
    high = np.minimum(low + 1, 126)
    down, up = m - _MAGNITUDES[low], _MAGNITUDES[high] - m
    pick = np.where((up < down) | ((up == down) & (low % 2 == 1)), high, low)
    return np.where(np.isnan(m), 127, pick + 128 * np.signbit(v)).astype(np.uint8)


def quantize(x):
    """(bytes [r, 128 blocks], scale bytes [r, blocks]) of rows x."""
    r, k = x.shape
    blocks = -(-k // 128)
    x = np.concatenate([x.astype(np.float64), np.zeros((r, 128 * blocks - k))], 1).reshape(r, blocks, 128)
    x = np.where(np.isfinite(x), x, np.nan)
    largest = np.nanmax(np.where(np.isnan(x), 0, np.abs(x)), 2)
    m, e = np.frexp(largest)  # 448 = 0.875 x 2^9
    e = np.where(largest > 0, np.maximum(e - 9 + (m > 0.875), -127), 0)
    return to_bytes(np.ldexp(x, -e[:, :, None])).reshape(r, -1), (e + 127).astype(np.uint8)


def values(data, scales, k):
    """f64 rows of k that bytes and scales stand for."""
    r, blocks = data.shape[0], -(-k // 128)
    v = E4M3[data[:, :128 * blocks]].reshape(r, blocks, 128)
    return np.ldexp(v, scales[:, :blocks, None].astype(int) - 127).reshape(r, -1)[:, :k]


def weights(w, taps):
    """f64 values of weights (taps c) x n in 8 bits."""
    c, n = w.shape[0] // taps, w.shape[1]
    rows = np.ascontiguousarray(w.reshape(taps, c, n).transpose(0, 2, 1).reshape(taps * n, c))
    return values(*quantize(rows), c).reshape(taps, n, c).transpose(0, 2, 1).reshape(taps * c, n)


def patches(x, images, height, width, step):
    """Rows [images oh ow, 9 c] of the zero-padded 3 x 3 taps of pixels x."""
    c = x.shape[1]
    p = np.zeros((images, height + 2, width + 2, c))
    p[:, 1:-1, 1:-1] = x.reshape(images, height, width, c)
    return np.concatenate([p[:, dy:dy + height:step, dx:dx + width:step].reshape(-1, c)
                           for dy in range(3) for dx in range(3)], 1)


def activate(v, act):
    import math

    if act == "relu":
        return np.where(v < 0, 0, v)
    if act == "gelu":
        return 0.5 * v * (1 + np.vectorize(math.erf)(v / math.sqrt(2)))
    if act == "sigmoid":
        return 1 / (1 + np.exp(-v))
    return v / (1 + np.exp(-v)) if act == "silu" else v


# The steepest slope of each activation (what an error before it can grow by).
SLOPE = {"none": 1.0, "relu": 1.0, "sigmoid": 0.25, "gelu": 1.13, "silu": 1.1}


def group_norm(x, images, groups, gamma, beta, eps, act):
    """(y, the normalised values' magnitude before gamma): f64 rows."""
    rows, c = x.shape
    v = x.astype(np.float64).reshape(images, rows // images, groups, c // groups)
    mean = v.mean((1, 3), keepdims=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdims=True)
    n = ((v - mean) / np.sqrt(var + eps)).reshape(rows, c)
    # How far a mean or deviation that is off by one part in 2^24 moves a value.
    reach = (np.abs(mean) + np.abs(v)) / np.sqrt(var + eps)
    g = 1.0 if gamma is None else gamma.astype(np.float64)
    b = 0.0 if beta is None else beta.astype(np.float64)
    return activate(n * g + b, act), reach.reshape(rows, c) * np.abs(g) + np.abs(b)

"""8-bit layers, restated in NumPy from their formulas (posehip/w8a8.py): bit-exact forms (every f32 rounding where the
definition has one) and the same in 64 bits without any."""
import numpy as np

TINY = np.float32(2.0 ** -126)


def quantize_rows(x):
    """x [M,K] of any float type (exact in f64) -> (q int8, scale f32 [M])."""
    x = np.asarray(x, np.float64)
    amax = np.abs(x).max(axis=1)
    ok = np.isfinite(amax)
    with np.errstate(invalid="ignore"):
        # f64 division then rounding to f32 = the f32 quotient (53 >= 2 * 24 + 2 bits)
        s = np.maximum((np.where(ok, amax, 0.0) / 127.0).astype(np.float32), TINY)
        # two numbers of 24 bits have no quotient within 2^-53 of a border k + 1/2 but on it
        q = np.rint(np.where(ok[:, None], x, 0.0) / s.astype(np.float64)[:, None])
    return q.astype(np.int8), np.where(ok, s, np.float32(np.nan)).astype(np.float32)


def sums(q, w):
    """exact: every product and partial sum is below 2^53"""
    return np.asarray(q, np.float64) @ np.asarray(w, np.float64).T


def act32(y, act, slope):
    if act == "relu":
        return np.where(y < 0, np.float32(0), y)
    if act == "prelu":
        return np.where(y < 0, y * np.asarray(slope, np.float32)[None], y)
    return y


def matmul(q, s, w, ws, bias=None, act="none", slope=None):
    """-> f32 [M,N], each operation rounded as the definition has it"""
    with np.errstate(invalid="ignore", over="ignore"):
        y = sums(q, w).astype(np.float32) * np.asarray(ws, np.float32)[None] * np.asarray(s, np.float32)[:, None]
        if bias is not None:
            y = y + np.asarray(bias, np.float32)[None]
        return act32(y, act, slope).astype(np.float32)


def linear(x, w, ws, bias=None, act="none", slope=None):
    return matmul(*quantize_rows(x), w, ws, bias, act, slope)


def feed_forward(x, l1, l2):
    """l1, l2: (w, ws, bias, act, slope)"""
    return linear(linear(x, *l1), *l2)


def matmul64(q, s, w, ws, bias=None, act="none", slope=None):
    """(y, sum of the magnitudes that the additions and products pass through) in 64 bits"""
    y = sums(q, w) * np.asarray(ws, np.float64)[None] * np.asarray(s, np.float64)[:, None]
    mag = np.abs(y)
    if bias is not None:
        y = y + np.asarray(bias, np.float64)[None]
        mag = mag + np.abs(np.asarray(bias, np.float64))[None]
    if act == "relu":
        y = np.maximum(y, 0)
    elif act == "prelu":
        y = np.where(y < 0, y * np.asarray(slope, np.float64)[None], y)
    return y, mag

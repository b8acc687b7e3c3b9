"""Microscaled 4-bit floating point and the root-mean-square norm from their definitions in 64 bits: what the tests of those
operators compare with."""
import numpy as np

BLOCK = 32
VALUES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantize(x):
    """(codes uint8 [rows][cols], scale bytes uint8 [rows][cols / 32]) of floats [rows][cols]."""
    x = np.asarray(x, np.float64)
    rows, cols = x.shape
    b = x.reshape(rows, cols // BLOCK, BLOCK)
    bad = ~np.isfinite(b).all(2)
    b = np.where(bad[:, :, None], 0.0, b)
    top = np.abs(b).max(2)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)  # floor(log2(top)) - 2
    e = np.maximum(e, -127)
    z = np.abs(b) * 2.0 ** -e[:, :, None].astype(np.float64)
    hi = np.clip(np.searchsorted(VALUES, z), 1, 7)
    lo = hi - 1
    down, up = z - VALUES[lo], VALUES[hi] - z
    pick = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))  # halves to the even code
    codes = (pick + 8 * np.signbit(b)).astype(np.uint8)
    codes[bad] = 0
    return codes.reshape(rows, cols), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, scales):
    """What codes and scale bytes stand for, f64; the byte 255 is NaN."""
    v = VALUES[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return v * np.repeat(s, BLOCK, 1)


def blocks(codes, scales):
    """GGUF's bytes: the scale, then byte i with element i in the low half and element i + 16 in the high one."""
    rows, cols = codes.shape
    c = codes.reshape(rows, cols // BLOCK, BLOCK)
    return np.concatenate([scales[:, :, None], c[:, :, :16] | c[:, :, 16:] << 4], 2)


def random_matrix(rng, rows, cols, spread=3):
    """All sixteen codes, the scales over 2 * spread powers of two."""
    return rng.integers(0, 16, (rows, cols), dtype=np.uint8), rng.integers(120 - spread, 120 + spread, (rows, cols // BLOCK), dtype=np.uint8)


def product(codes, scales, x):
    """(y, room): x W^T in 64 bits over x quantized, and how far the kernels' may be.  Within a block products are whole quarters of at
    most 36 under one power of two: eight of them at a time are exact.  Every such sum meets the running one with an error of at most a
    step of its last place, 2^-23 of the sum of magnitudes; wavefronts' sums and parts meet in fewer than 24 more."""
    a, w = values(*quantize(x)), values(codes, scales)
    with np.errstate(invalid="ignore"):
        return a @ w.T, (w.shape[1] / 8 + 24) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)


def norm(x, residual, weight, eps, rounded):
    """(h, y): h in 64 bits holding numbers of the type that `rounded` rounds to, y f32."""
    h = np.asarray(x, np.float64)
    if residual is not None:
        h = rounded((np.asarray(x, np.float32) + np.asarray(residual, np.float32)).astype(np.float32))
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        r = (1.0 / np.sqrt((h * h).sum(1, keepdims=True) / h.shape[1] + eps)).astype(np.float32)
        y = (h.astype(np.float32) * r).astype(np.float32)
        return h, y if weight is None else (y * np.asarray(weight, np.float32)).astype(np.float32)

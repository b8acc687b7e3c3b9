"""Weights in 8-bit floating point with a scale for each block of 128 x 128, and routing by a rule, from their definitions in
64 bits: what the tests of those operators compare with."""
import numpy as np

BLOCK = 128


def e4m3_values():
    """The value of each of E4M3's 256 codes: a sign, four bits of exponent (bias 7), three of mantissa; 0x7f and 0xff NaN."""
    v = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v[c] = np.nan if c & 0x7f == 0x7f else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        if c & 0x80:
            v[c] = -v[c]
    return v


VALUES = e4m3_values()


def to_e4m3(z):
    """Values of |z| <= 448 to the nearest value of E4M3, halves to the even code."""
    grid = VALUES[:127]  # ascending, 0 .. 448
    a = np.abs(z)
    hi = np.clip(np.searchsorted(grid, a), 1, 126)
    lo = hi - 1
    down, up = a - grid[lo], grid[hi] - a
    pick = np.where(up < down, hi, np.where(up > down, lo, np.where(hi % 2 == 0, hi, lo)))
    return np.copysign(grid[pick], z)


def quantize(x):
    """The values that activations [rows][cols] f32 have once quantized (f64)."""
    x = np.asarray(x, np.float64)
    out = np.empty_like(x)
    for k in range(0, x.shape[1], BLOCK):
        v = x[:, k:k + BLOCK]
        fine = np.isfinite(v)
        top = np.where(fine, np.abs(v), 0.0).max(1, keepdims=True)
        e = np.full(top.shape, -100.0)
        while (top > 448.0 * 2.0 ** e).any():
            e = np.where(top > 448.0 * 2.0 ** e, e + 1, e)
        with np.errstate(invalid="ignore"):
            out[:, k:k + BLOCK] = np.where(fine, to_e4m3(np.where(fine, v, 0.0) * 2.0 ** -e) * 2.0 ** e, np.nan)
    return np.clip(out, -240 * 2.0 ** 120, 240 * 2.0 ** 120)  # (the next code's value is no float)


def expand(scales, rows, cols):
    """One matrix's scales [row blocks][blocks] as [rows][cols]."""
    return np.repeat(np.repeat(np.asarray(scales, np.float64), BLOCK, 0)[:rows], BLOCK, 1)[:, :cols]


def dequant(codes, scales):
    """codes [rows][cols] uint8 of one matrix, f64."""
    return VALUES[codes] * expand(scales, *codes.shape)


def random_matrix(rng, rows, cols, matrices=1):
    """(codes [matrices][rows][cols], scales): all finite codes, the scales over a few powers of two."""
    codes = rng.integers(0, 127, (matrices, rows, cols), dtype=np.uint8) | rng.integers(0, 2, (matrices, rows, cols), dtype=np.uint8) << 7
    blocks = (matrices, -(-rows // BLOCK), -(-cols // BLOCK))
    scales = (rng.uniform(0.5, 2.0, blocks) * 2.0 ** rng.integers(-9, -6, blocks)).astype(np.float32)
    return codes, scales


def product(codes, scales, x):
    """(y, room): x W^T in 64 bits, and how far f32 sums may be from it.  A matrix-core step adds 128 exact products: at most
    128 roundings of partial sums; every block's result is then multiplied and added in one rounding, at most `blocks` of them
    in a row, and eight wavefronts' sums meet in seven more; each rounding is 2^-24 of at most the sum of magnitudes."""
    a, w = quantize(x), dequant(codes, scales)
    return a @ w.T, (128 + w.shape[1] / BLOCK + 9) * 2.0 ** -24 * (np.abs(a) @ np.abs(w).T)


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_best=1, norm=True, scale=1.0):
    """ids and weights (f64) of each row, by sorting; equal values to the lower index."""
    l = np.asarray(logits, np.float64)
    batch, n = l.shape
    ids, weights = np.full((batch, k), -1, np.int32), np.zeros((batch, k))
    for b in range(batch):
        live = np.array([v > -np.inf for v in l[b]])  # (NaN: not)
        p = np.zeros(n)
        if live.any():
            if score == "sigmoid":
                p[live] = 1 / (1 + np.exp(-l[b][live]))
            else:
                top = l[b][live].max()
                e = np.where(l[b][live] == top, 1.0, np.exp(l[b][live] - top) if np.isfinite(top) else 0.0)
                p[live] = e / e.sum()
        c = p + (np.asarray(bias, np.float64) if bias is not None else 0.0)
        c[~live] = -np.inf
        size = n // groups
        if groups > 1:
            value = []
            for g in range(groups):
                best = sorted((v for v in c[g * size:(g + 1) * size] if v > -np.inf), reverse=True)[:group_best]
                value.append(sum(best) if best else -np.inf)
            used = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
            c = np.where(np.isin(np.arange(n) // size, used), c, -np.inf)
        chosen = [i for i in sorted(range(n), key=lambda i: (-c[i], i))[:k] if c[i] > -np.inf]
        w = p[chosen]
        if norm:
            w = w / w.sum() if w.sum() > 0 else w * 0
        ids[b, :len(chosen)] = chosen
        weights[b, :len(chosen)] = w * np.float64(np.float32(scale))
    return ids, weights

"""The 8-bit cache format and the attention over it in 64 bits (numpy), from their definitions.

A block of 32 dims of one token's head, largest magnitude A, is held as codes and an exponent byte e + 127,
e the smallest integer with M * 2^e >= A within the format's limits, M its largest code; codes are x * 2^-e
rounded to the nearest, ties to even, cut at +-M. A block with a NaN or an infinity has the byte 255.
"""
import numpy as np

BLOCK = 32
FORMATS = {"int8": (127.0, -24, 9), "fp8": (448.0, -15, 7)}


def code_values(fmt):
    """The value of each of the 256 codes, before its exponent."""
    c = np.arange(256)
    if fmt == "int8":
        return np.where(c < 128, c, c - 256).astype(np.float64)
    e, m = (c >> 3) & 15, (c & 7) / 8.0
    v = np.where(e == 0, m * 2.0 ** -6, (1 + m) * 2.0 ** (e - 7.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


def quantise(x, fmt):
    """fp64 rows [..., D] -> (values as held [..., D], exponent bytes [..., ceil(D / 32)])."""
    top, lo, hi = FORMATS[fmt]
    grid = np.unique(code_values(fmt)[np.isfinite(code_values(fmt))])
    grid = grid[np.abs(grid) <= top]
    nb = -(-x.shape[-1] // BLOCK)
    out, exps = np.empty(x.shape), np.empty(x.shape[:-1] + (nb,), dtype=np.uint8)
    for i in range(nb):
        y = x[..., BLOCK * i:BLOCK * (i + 1)]
        with np.errstate(invalid="ignore"):
            big = np.abs(y).max(-1)
        bad = ~np.isfinite(big)
        e = np.full(big.shape, lo)
        for p in range(lo, hi):
            e = np.where(np.where(bad, 0, big) > top * 2.0 ** p, p + 1, e)
        z = np.clip(np.where(bad[..., None], 0, y) / 2.0 ** e[..., None], -top, top)
        # the two neighbouring numbers of the grid; of two equally near ones that with an even last bit
        up = np.clip(np.searchsorted(grid, z, side="left"), 0, len(grid) - 1)
        down = np.maximum(up - (grid[up] > z), 0)
        du, dd = grid[up] - z, z - grid[down]
        step = grid[up] - grid[down]
        even = np.where(step > 0, np.mod(np.rint(grid[up] / np.where(step > 0, step, 1)), 2) == 0, True)
        z = np.where((du < dd) | ((du == dd) & even), grid[up], grid[down])
        out[..., BLOCK * i:BLOCK * (i + 1)] = np.where(bad[..., None], np.nan, z * 2.0 ** e[..., None])
        exps[..., i] = np.where(bad, 255, e + 127)
    return out, exps


def held(codes, exps, fmt):
    """The values of codes uint8 [..., D] under exponent bytes [..., blocks]."""
    s = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    return code_values(fmt)[codes] * np.repeat(s, BLOCK, -1)[..., :codes.shape[-1]]


def attend(q, k, v, scale):
    """softmax(scale q k^T) v of one query row [D] over keys [T, D]; NaN without a key.

    Returns (out, spread): spread is what an error in the weights is measured by, sum(p |v|) per dim."""
    if len(k) == 0:
        return np.full(v.shape[-1], np.nan), np.zeros(v.shape[-1])
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v)

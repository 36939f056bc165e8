"""Rows of 4-bit values (GQ_KV_E2M1) by their definition, in 64 bits: what a block of 16 numbers
becomes, and what its codes and scale stand for."""
import numpy as np

CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
SCALES = np.array([(8 + f) * 2.0 ** (e - 10) if e else f * 2.0 ** -9 for e in range(16) for f in range(8)][:127])  # e4m3


def nearest(y, grid):
    """Index of the nearest of the ascending grid; between two the even index; past the end the last."""
    hi = np.clip(np.searchsorted(grid, y), 1, len(grid) - 1)
    lo = hi - 1
    up, down = grid[hi] - y, y - grid[lo]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


def encode(v, scale):
    """Rows [..., head_dim] f32 -> [..., head_dim / 16 * 9] uint8. (A quotient of two numbers of 24 and
    of 4 bits is a tie or at least 2^-28 of itself away from one: 64 bits tell them apart.)"""
    x = (np.asarray(v, np.float32) * np.float32(1.0 / np.float32(scale))).astype(np.float64)
    x = x.reshape(*x.shape[:-1], x.shape[-1] // 16, 16)
    a = np.abs(x)
    top = a.max(-1)
    with np.errstate(invalid="ignore"):
        s = nearest(np.minimum(top / 6, 448.0), SCALES)
    s[np.isnan(top)] = 127
    div = np.where((s == 0) | (s == 127), np.inf, np.append(SCALES, np.nan)[s])[..., None]
    with np.errstate(invalid="ignore"):
        y = np.where(np.isinf(a), np.where(np.isinf(div), 0.0, 6.0), a / div)
    c = nearest(np.minimum(np.nan_to_num(y, nan=0.0), 6.0), CODES) + 8 * np.signbit(x)
    c = c.reshape(*c.shape[:-2], c.shape[-2] * 8, 2).astype(np.uint8)
    return np.concatenate([c[..., 0] | (c[..., 1] << 4), s.astype(np.uint8)], -1)


def decode(rows, scale=1.0):
    """[..., head_dim / 16 * 9] uint8 -> the values [..., head_dim], f64."""
    d = rows.shape[-1] // 9 * 16
    packed, s = rows[..., :d // 2], rows[..., d // 2:]
    c = np.stack([packed & 15, packed >> 4], -1).reshape(*rows.shape[:-1], d)
    v = np.where(c >= 8, -1.0, 1.0) * CODES[c & 7]
    table = np.concatenate([SCALES, [np.nan], -SCALES, [np.nan]])
    return v * np.repeat(table[s], 16, -1) * float(scale)

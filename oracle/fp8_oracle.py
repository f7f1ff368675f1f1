"""64-bit restatement of the block-scaled 8-bit floating point operators and of counter-based dropout (numpy, from the
definitions; shares nothing with the package)."""

from __future__ import annotations

import numpy as np

#: largest magnitude, mantissa bits, exponent of the smallest normal number
FORMATS = {"e4m3": (448.0, 3, -6), "e5m2": (57344.0, 2, -14)}


def philox4x32_10(counter, key):
    """Philox4x32 with ten rounds on python integers: counter of four words, key of two (for known-answer tests)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(elements, p: float, seed: int, offset: int):
    """Truth value for each element number: its 16 bits are >= round(p 65536)."""
    elements = np.asarray(elements, dtype=np.uint64)
    g = elements >> np.uint64(3)
    low = np.uint64(0xFFFFFFFF)
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    c = [g & low, g >> np.uint64(32), np.full_like(g, offset & 0xFFFFFFFF), np.full_like(g, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    words = np.stack(c, axis=-1)
    place = (elements & np.uint64(7)).astype(np.int64)
    word = np.take_along_axis(words, (place >> 1)[..., None], axis=-1)[..., 0]
    half = (word >> ((place & 1) * 16).astype(np.uint64)) & np.uint64(0xFFFF)
    return half >= np.uint64(round(p * 65536))


def keep_mask(shape, p, seed, offset):
    n = int(np.prod(shape))
    return kept(np.arange(n, dtype=np.uint64), p, seed, offset).reshape(shape)


def round_to_format(v, fmt):
    """Nearest number of the format, ties to even; |v| is at most the largest one."""
    _, mbits, least = FORMATS[fmt]
    a = np.abs(v)
    e = np.maximum(np.frexp(np.where(a > 0, a, 1.0))[1] - 1, least)
    unit = np.exp2(e.astype(np.float64) - mbits)
    return np.rint(v / unit) * unit


def quantise(x, fmt="e4m3", block_rows=1):
    """(numbers [R, C] in 64 bits, scales [ceil(R / block_rows), ceil(C / 128)])."""
    x = np.asarray(x, dtype=np.float64)
    R, C = x.shape
    nr, nc = -(-R // block_rows), -(-C // 128)
    q, s = np.zeros((R, C)), np.zeros((nr, nc))
    for i in range(nr):
        for j in range(nc):
            blk = np.s_[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            v = x[blk]
            if not np.isfinite(v).all():
                q[blk], s[i, j] = np.nan, np.nan
                continue
            a = np.abs(v).max()
            e = -126
            if a > 0:
                m, ex = np.frexp(a)                              # a = m 2^ex, m in [0.5, 1)
                mf, ef = np.frexp(FORMATS[fmt][0])
                e = max(int(ex - ef + (m > mf)), -126)
            s[i, j] = 2.0 ** e
            q[blk] = round_to_format(v / s[i, j], fmt)
    return q, s


def dequantise(q, s):
    rows = 1 if s.shape[0] == q.shape[0] else 128
    return np.asarray(q, np.float64) * np.repeat(np.repeat(s, rows, 0)[:q.shape[0]], 128, 1)[:, :q.shape[1]]


def product(a, sa, b, sb, bias=None, alpha=1.0):
    """(y, sum of magnitudes): the second bounds what an fp32 sum may be off by."""
    da, db = dequantise(a, sa), dequantise(b, sb)
    y, mag = alpha * (da @ db.T), abs(alpha) * (np.abs(da) @ np.abs(db).T)
    if bias is not None:
        y, mag = y + np.asarray(bias, np.float64), mag + np.abs(np.asarray(bias, np.float64))
    return y, mag

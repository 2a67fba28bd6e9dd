"""Philox4x32-10 in numpy, for the tests of dropout: words of counters (column // 4, row, offset low, offset high) under a 64-bit seed."""
import numpy as np

LOW = np.uint64(0xFFFFFFFF)
HALF = np.uint64(32)


def rounds(counter, key):
    """Four arrays of words (uint64 below 2^32) from a counter of four and a key of two."""
    a, b, c, d = (np.asarray(x, dtype=np.uint64) for x in counter)
    k, m = int(key[0]), int(key[1])
    for _ in range(10):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (q >> HALF) ^ b ^ np.uint64(k), q & LOW, (p >> HALF) ^ d ^ np.uint64(m), p & LOW
        k, m = (k + 0x9E3779B9) & 0xFFFFFFFF, (m + 0xBB67AE85) & 0xFFFFFFFF
    return a, b, c, d


def kept(rows, cols, p, seed, offset, first_row=0):
    """The mask of dropout: [rows, cols] truth values."""
    group, row = np.meshgrid(np.arange((cols + 3) // 4, dtype=np.uint64), np.arange(first_row, first_row + rows, dtype=np.uint64))
    lo, hi = np.full_like(group, offset & 0xFFFFFFFF), np.full_like(group, offset >> 32)
    seed &= 0xFFFFFFFFFFFFFFFF
    words = np.stack(rounds((group, row, lo, hi), (seed & 0xFFFFFFFF, seed >> 32)), -1).reshape(rows, -1)[:, :cols]
    return words >= np.uint64(int(p * 2.0 ** 32 + 0.5))


def grown(p):
    """What a kept value is multiplied by."""
    return 2.0 ** 32 / (2 ** 32 - int(p * 2.0 ** 32 + 0.5))

"""Philox4x32 with ten rounds (Salmon et al., Parallel random numbers: as easy as 1, 2, 3,
SC 2011), in numpy's 64-bit whole numbers."""
import numpy as np


def philox(counter, key):
    """Four words of 32 bits from four (arrays) and two."""
    a, b, c, d = np.broadcast_arrays(*(np.asarray(w, dtype=np.uint64) for w in counter))
    k0, k1 = (np.uint64(k) for k in key)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (q >> half) ^ b ^ k0, q & low, (p >> half) ^ d ^ k1, p & low
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & low, (k1 + np.uint64(0xBB67AE85)) & low
    return a, b, c, d


def numbers(rows, cols, seed, step, first_row=0):
    """[rows, cols] numbers of a dropout call."""
    blocks = -(-cols // 4)
    words = philox((np.arange(blocks), (np.arange(rows) + first_row)[:, None], step & 0xFFFFFFFF, step >> 32),
                   (seed & 0xFFFFFFFF, seed >> 32))
    return np.stack(words, 2).reshape(rows, 4 * blocks)[:, :cols]

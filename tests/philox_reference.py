"""Philox4x32 with 7 rounds (Salmon, Moraes, Dror and Shaw 2011) in numpy's unsigned integers,
and the dropout mask formed from it: what the HIP kernels are tested against."""
import numpy as np


def philox4x32(counter, key, rounds):
    """counter: four uint64 arrays of 32-bit words, key: two ints; four arrays of 32-bit words."""
    lo, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = [np.asarray(w, np.uint64) for w in counter], list(key)
    for _ in range(rounds):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> sh) ^ c[1] ^ np.uint64(k[0]), p1 & lo, (p0 >> sh) ^ c[3] ^ np.uint64(k[1]), p0 & lo]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(n, p, seed, offset, first=0):
    """Whether each of n elements from element 8 first on is kept: 16 bits of the stream below
    round((1 - p) 65536)."""
    j = np.arange(first, first - (-n // 8), dtype=np.uint64)
    lo = np.uint64(0xFFFFFFFF)
    words = philox4x32((j & lo, j >> np.uint64(32), np.full_like(j, offset & 0xFFFFFFFF), np.full_like(j, offset >> 32)),
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF), 7)
    return np.stack(words, 1).astype("<u4").reshape(-1).view("<u2")[:n] < round((1.0 - p) * 65536)

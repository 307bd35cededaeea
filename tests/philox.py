"""Philox4x32-10 in numpy, for the tests of dropout: written from the published description (Salmon et al. 2011)."""
import numpy as np


def words(first, count, seed, counter=None, key=None):
    """Words first .. first + count - 1 of the stream of `seed`: word i is word i % 4 of counter (i / 4, 0, 0)."""
    lo, n = first // 4, (first + count + 3) // 4 - first // 4
    block = np.arange(lo, lo + n, dtype=np.uint64)
    mask = np.uint64(0xffffffff)
    c = [block & mask, block >> np.uint64(32), np.zeros_like(block), np.zeros_like(block)] if counter is None else [np.full(n, v, dtype=np.uint64) for v in counter]
    k = [seed & 0xffffffff, seed >> 32 & 0xffffffff] if key is None else list(key)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)  # (32 x 32 bits fit 64)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [k[0] + 0x9E3779B9 & 0xffffffff, k[1] + 0xBB67AE85 & 0xffffffff]
    return np.stack(c, 1).reshape(-1)[first - 4 * lo:][:count]


def kept(first, count, p, seed):
    return words(first, count, seed) >= np.uint64(round(p * 2 ** 32))

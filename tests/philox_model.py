"""Philox-4x32-10 (Salmon et al. 2011) in numpy: the decisions of dropout by counter."""
import numpy as np


def words(seed, first, n):
    """Words of elements first .. first + n - 1: word i % 4 of counter (i // 4, 0) under the seed's halves."""
    block0, block1 = first // 4, (first + n + 3) // 4
    counter = np.arange(block0, block1, dtype=np.uint64)
    mask = np.uint64(0xFFFFFFFF)
    c = [counter & mask, counter >> np.uint64(32), np.zeros_like(counter), np.zeros_like(counter)]
    k = [seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & mask, (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & mask]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[first - 4 * block0:][:n].astype(np.uint32)


def keep(seed, p, n):
    """Which of n elements stay."""
    threshold = min(max(int(p * 2 ** 32), 1), 2 ** 32 - 1) if p > 0 else 0
    return words(seed, 0, n) >= np.uint32(threshold)

"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011) in numpy."""
import numpy as np

W = np.uint64(0xFFFFFFFF)
S = np.uint64(32)


def philox(c, k):
    """c (4, n) uint64 words, k (k0, k1) -> (4, n) words"""
    k0, k1 = k
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = np.stack([(b >> S) ^ c[1] ^ np.uint64(k0), b & W, (a >> S) ^ c[3] ^ np.uint64(k1), a & W])
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def pieces(i, seed, offset):
    """the 16-bit pieces of elements i (int array)"""
    i = np.asarray(i).astype(np.uint64)
    b = i >> np.uint64(3)
    off = np.full_like(b, offset)
    w = philox(np.stack([b & W, b >> S, off & W, off >> S]), (seed & 0xFFFFFFFF, seed >> 32))
    e = (i & np.uint64(7)).astype(np.int64)
    return (w[e >> 1, np.arange(i.size)] >> ((e & 1) * 16).astype(np.uint64)) & np.uint64(0xFFFF)

"""Philox 4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011) in Python's integers and in numpy, and
the dropout that the library makes of it: 16 bits a value, eight values a counter."""
import numpy as np


def words(counter, key):
    """Four words of one counter, in Python's integers."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p, q = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(q >> 32) ^ c[1] ^ k[0], q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k[1], p & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def bits(first, count, seed, offset):
    """The 16 bits of the values first .. first + count (first: a multiple of 8)."""
    j = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [j & low, j >> half, np.full_like(j, offset & 0xFFFFFFFF), np.full_like(j, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ np.uint64(k0), q & low, (p >> half) ^ c[3] ^ np.uint64(k1), p & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack([np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], 1) for w in c], 1).reshape(-1)[:count].astype(np.int64)


def share(rate):
    return int(rate * 65536 + 0.5)


def keep(first, count, rate, seed, offset=0):
    return bits(first, count, seed, offset) >= share(rate)

"""The oracle of dropout's mask, element by element in Python's and numpy's whole numbers:
Philox4x32 (Salmon, Moraes, Dror, Shaw, SC 2011)."""
import numpy as np

M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
LOW = np.uint64(0xffffffff)


def philox(counter, key, rounds):
    """One block, in Python's numbers."""
    c0, c1, c2, c3 = counter
    k0, k1 = key
    for _ in range(rounds):
        a, b = c0 * M0, c2 * M1
        c0, c1, c2, c3 = (b >> 32) ^ c1 ^ k0, b & 0xffffffff, (a >> 32) ^ c3 ^ k1, a & 0xffffffff
        k0, k1 = (k0 + W0) & 0xffffffff, (k1 + W1) & 0xffffffff
    return c0, c1, c2, c3


def bits(count, seed, site):
    """The sixteen random bits of `count` elements."""
    group = np.arange((count + 7) // 8, dtype=np.uint64)
    c0, c1 = group & LOW, group >> np.uint64(32)
    c2, c3 = np.full_like(group, site), np.zeros_like(group)
    key = seed % 2 ** 64
    for r in range(7):
        k0 = np.uint64((key % 2 ** 32 + r * W0) % 2 ** 32)
        k1 = np.uint64((key // 2 ** 32 + r * W1) % 2 ** 32)
        a, b = c0 * np.uint64(M0), c2 * np.uint64(M1)
        c0, c1, c2, c3 = b >> np.uint64(32) ^ c1 ^ k0, b & LOW, a >> np.uint64(32) ^ c3 ^ k1, a & LOW
    words = np.stack([c0, c1, c2, c3], axis=1)
    halves = np.stack([words & np.uint64(0xffff), words >> np.uint64(16)], axis=2)
    return halves.reshape(-1)[:count]


def mask(shape, p, seed, site=0):
    """(truth values of what is kept, the factor of what is)"""
    below = round(65536 * p)
    count = int(np.prod(shape))
    return (bits(count, seed, site) >= below).reshape(shape), 0.0 if below == 65536 else 65536 / (65536 - below)

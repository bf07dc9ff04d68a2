"""64-bit restatements of the residual-block operators (include/dcn.h), for the tests only:
Philox4x32-10 draws, dropout, block norms with their gradients by torch's float64 autograd,
and 8-bit block rounding. Written from the definitions, on the CPU."""
from __future__ import annotations

import numpy as np
import torch

M32 = 0xFFFFFFFF


def philox4x32_10(ctr, key):
    """Four words of Philox4x32-10 for one counter (4 words) and key (2 words), Python ints."""
    x, k = list(ctr), list(key)
    for _ in range(10):
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        x = [(p1 >> 32) ^ x[1] ^ k[0], p1 & M32, (p0 >> 32) ^ x[3] ^ k[1], p0 & M32]
        k = [(k[0] + 0x9E3779B9) & M32, (k[1] + 0xBB67AE85) & M32]
    return x


def draws(first, n, seed, offset):
    """The 16-bit draws of elements first .. first + n - 1."""
    b0 = first >> 3
    i = np.arange(b0, (first + n + 7) // 8, dtype=np.uint64)
    m, s = np.uint64(M32), np.uint64(32)
    x = [i & m, i >> s, np.full_like(i, offset & M32), np.full_like(i, (offset >> 32) & M32)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        p0, p1 = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(p1 >> s) ^ x[1] ^ np.uint64(k0), p1 & m, (p0 >> s) ^ x[3] ^ np.uint64(k1), p0 & m]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    u = np.stack([h for w in x for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return u.reshape(-1)[first - 8 * b0:][:n].astype(np.int64)


def drop_factor(n, group, p, seed, offset):
    """0 or 65536 / (65536 - T) per element, float64."""
    t = int(np.floor(p * 65536 + 0.5))
    nd = -(-n // group)
    f = np.where(draws(0, nd, seed, offset) < t, 0.0, 65536.0 / max(65536 - t, 1))
    return np.repeat(f, group)[:n]

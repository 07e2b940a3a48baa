"""The dropout operators' random numbers in numpy: Philox4x32-10 from its published definition."""

from __future__ import annotations

import numpy as np

_LOW = np.uint64(0xFFFFFFFF)


def philox(counters: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """counters: [n, 4] 32-bit words; returns [n, 4] uint32."""
    c = [counters[:, i].astype(np.uint64) & _LOW for i in range(4)]
    k = list(key)
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), q & _LOW,
             (p >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p & _LOW]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return np.stack(c, 1).astype(np.uint32)


def numbers(cells: int, seed: int, subsequence: int = 0, first: int = 0) -> np.ndarray:
    """The 16-bit numbers of elements first .. first + cells - 1 (first a multiple of 8)."""
    g = np.arange(first // 8, first // 8 + (cells + 7) // 8, dtype=np.uint64)
    s = np.full_like(g, subsequence % 2**32), np.full_like(g, subsequence >> 32)
    words = philox(np.stack([g & _LOW, g >> np.uint64(32), *s], 1), (seed % 2**32, seed >> 32))
    halves = np.stack([words & np.uint32(0xFFFF), words >> np.uint32(16)], 2)
    return halves.reshape(-1)[:cells].astype(np.int64)


def factors(cells: int, p: float, seed: int, subsequence: int = 0) -> np.ndarray:
    """What each element is multiplied by, in 64 bits."""
    cut = int(p * 65536 + 0.5)
    if cut == 65536:
        return np.zeros(cells)
    return (numbers(cells, seed, subsequence) >= cut) * (65536.0 / (65536 - cut))

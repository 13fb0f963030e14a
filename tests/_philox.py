"""Which entries dropout keeps, in numpy from the generator's definition."""

import numpy as np
import torch


def philox(ctr, seed):
    """Philox4x32-10: ctr [..., 4] (uint64 arrays of 32-bit numbers) under a 64-bit key."""
    m32 = np.uint64(0xFFFFFFFF)
    c = [ctr[..., i].astype(np.uint64) for i in range(4)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        hi0, lo0, hi1, lo1 = p0 >> np.uint64(32), p0 & m32, p1 >> np.uint64(32), p1 & m32
        c = [hi1 ^ c[1] ^ np.uint64(k0), lo1, hi0 ^ c[3] ^ np.uint64(k1), lo0]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, -1)


def keep(rows, cols, p, seed, offset):
    """(mask [rows, cols], the factor of what is kept)."""
    groups = -(-cols // 8)
    i = np.arange(rows * groups, dtype=np.uint64)
    offset %= 2 ** 64
    ctr = np.stack([i & np.uint64(0xFFFFFFFF), i >> np.uint64(32), np.full_like(i, offset & 0xFFFFFFFF),
                    np.full_like(i, offset >> 32)], -1)
    words = philox(ctr, seed % 2 ** 64)
    halves = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], -1).reshape(rows, groups * 8)[:, :cols]
    cut = round(p * 65536)
    return torch.from_numpy(halves >= np.uint64(cut)), (65536 / (65536 - cut) if cut < 65536 else 0.0)

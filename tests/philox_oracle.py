"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) in numpy, and the
dropout factor that the row operators make from it."""
import numpy as np
import torch

M32 = np.uint64(0xFFFFFFFF)
S32 = np.uint64(32)


def philox(c, k):
    """c: four uint64 arrays of 32-bit words, k: two words -> four arrays."""
    c = [np.asarray(w, dtype=np.uint64) for w in c]
    k = [np.uint64(w) for w in k]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> S32) ^ c[1] ^ k[0], p1 & M32, (p0 >> S32) ^ c[3] ^ k[1], p0 & M32]
        k = [(k[0] + np.uint64(0x9E3779B9)) & M32, (k[1] + np.uint64(0xBB67AE85)) & M32]
    return c


def factor_at(i, p, seed, offset):
    """The factor (0 or the scale) of the elements with the indices i (uint64 array), as float64."""
    i = np.asarray(i, dtype=np.uint64)
    block = i >> np.uint64(3)
    off = [np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    words = np.stack(philox([block & M32, block >> S32] + off, [seed & 0xFFFFFFFF, seed >> 32]))
    j = (i & np.uint64(7)).astype(np.int64)
    w = np.take_along_axis(words, (j >> 1)[None], axis=0)[0]
    bits = np.where(j & 1, w >> np.uint64(16), w & np.uint64(0xFFFF)).astype(np.int64)
    thr = int(p * 65536 + 0.5)
    return np.where(bits >= thr, 65536.0 / max(1, 65536 - thr), 0.0)


def factor(shape, p, seed, offset):
    """... of a whole tensor read row by row, as a float64 torch tensor on the CPU."""
    n = int(np.prod(shape))
    return torch.from_numpy(factor_at(np.arange(n, dtype=np.uint64), p, seed, offset)).reshape(shape)

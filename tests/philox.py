"""Philox4x32-10 in numpy, and dropout by it: the oracle of the tests."""

import numpy as np
import torch


def philox(counter, key):
    """Philox4x32-10 on uint32 counters [n, 4] and a key of two words."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k = [np.uint64(v) for v in key]
    low, shift = np.uint64(0xffffffff), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ k[0], b & low,
             (a >> shift) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + np.uint64(0x9E3779B9)) & low,
             (k[1] + np.uint64(0xBB67AE85)) & low]
    return np.stack(c, 1).astype(np.uint32)


def expected(x, p, seed, step):
    """dropout(x) and where it keeps, on the CPU."""
    n = x.numel()
    b = np.arange(-(-n // 8), dtype=np.uint64)
    low, shift = np.uint64(0xffffffff), np.uint64(32)
    counter = np.stack([b & low, b >> shift,
                        np.full_like(b, step & 0xffffffff),
                        np.full_like(b, step >> 32)], 1)
    words = philox(counter, (seed & 0xffffffff, seed >> 32))
    bits = words.view(np.uint16).reshape(-1)[:n].astype(np.int64)
    t = round(p * 65536)
    keep = torch.from_numpy(bits >= t).view(x.shape)
    scale = torch.tensor(65536 / (65536 - t), dtype=torch.float32)
    y = x.cpu().float() * scale
    return torch.where(keep, y, torch.zeros(())).to(x.dtype), keep

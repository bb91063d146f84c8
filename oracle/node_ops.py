"""Node-wise operators in float64: embedding and its gradient, residual dropout, the gated feed-forward block. No
counterpart in the reference; stated from the formulas."""

import math

import numpy as np
import torch


def embedding(ids, table, scale):
    """scale * table[ids]; rows of NaN for ids outside the table."""
    t = table.double()
    ok = (ids >= 0) & (ids < t.shape[0])
    out = t[ids.clamp(0, t.shape[0] - 1)] * scale
    return torch.where(ok.unsqueeze(-1), out, torch.full_like(out, math.nan))


def embedding_grad(grad, ids, rows, scale, padding=None):
    """(gradient of the table, the same sum of absolute values, tokens per row)."""
    ids, g = ids.reshape(-1), grad.double().reshape(-1, grad.shape[-1])
    live = (ids >= 0) & (ids < rows)
    if padding is not None:
        live &= ids != padding
    ids, g = ids[live], g[live]
    zero = torch.zeros(rows, g.shape[1], dtype=torch.float64)
    return (zero.index_add(0, ids, g) * scale, zero.index_add(0, ids, g.abs()) * abs(scale),
            torch.bincount(ids, minlength=rows))


def philox4x32(counter, key):
    """Ten rounds of Philox4x32 (Salmon et al., 2011): counter (n, 4) and key (2) of numbers below 2^32, as (n, 4)."""
    c = [np.asarray(counter)[:, k].astype(np.uint64) for k in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k0), b & low, (a >> half) ^ c[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def dropout_keep(n, p, seed, offset, first=0):
    """Which of the elements first .. first + n - 1 are kept."""
    b0 = first // 4
    blocks = np.arange(b0, (first + n + 3) // 4, dtype=np.uint64)
    offset, seed = offset % 2 ** 64, seed % 2 ** 64
    counter = np.stack([blocks & np.uint64(0xFFFFFFFF), blocks >> np.uint64(32),
                        np.full_like(blocks, offset & 0xFFFFFFFF), np.full_like(blocks, offset >> 32)], axis=1)
    words = philox4x32(counter, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)[first - 4 * b0:][:n]
    return torch.from_numpy(words >= math.floor(p * 2 ** 32))


def dropout_add(x, residual, p, seed, offset):
    keep = dropout_keep(x.numel(), p, seed, offset).view(x.shape)
    kept = torch.where(keep, x.double() / (1 - p) if p < 1 else x.double(), torch.zeros((), dtype=torch.float64))
    return kept if residual is None else residual.double() + kept

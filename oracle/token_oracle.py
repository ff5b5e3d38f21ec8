"""Numpy restatement, in 64 bits, of the token-embedding operators: scaled lookup, dropout by Philox4x32-10 (Salmon,
Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011), gradient of the table."""
import math

import numpy as np

_LOW = np.uint64(0xFFFFFFFF)
_32 = np.uint64(32)


def philox4x32(counter, key, rounds=10):
    """counter: four uint32-valued uint64 arrays (or numbers), key: two numbers -> four arrays of 32-bit words."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)  # (32 x 32 bits: no overflow)
        c = [(b >> _32) ^ c[1] ^ np.uint64(k[0]), b & _LOW, (a >> _32) ^ c[3] ^ np.uint64(k[1]), a & _LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def threshold(p):
    return math.floor(65536 * p + 0.5)


def factor(scale, p):
    t = threshold(p)
    return scale * 65536 / (65536 - t) if t < 65536 else 0.0


def kept(rows, dim, p, seed, offset):
    """[rows, dim] bool."""
    blocks = (dim + 7) // 8
    c0 = np.broadcast_to(np.arange(blocks, dtype=np.uint64), (rows, blocks))
    c1 = np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], (rows, blocks))
    words = philox4x32((c0, c1, offset & 0xFFFFFFFF, offset >> 32), (seed & 0xFFFFFFFF, seed >> 32))
    draws = np.stack([np.broadcast_to(w >> np.uint64(s), (rows, blocks)) & np.uint64(0xFFFF) for w in words for s in (0, 16)], axis=2)
    return draws.reshape(rows, blocks * 8)[:, :dim] >= np.uint64(threshold(p))


def dropped(x, scale=1.0, p=0.0, seed=0, offset=0):
    """float64 [rows, dim]; dropped values are zeros whatever they were."""
    x = np.asarray(x, dtype=np.float64)
    keep = kept(x.shape[0], x.shape[1], p, seed, offset) if threshold(p) else np.ones(x.shape, bool)
    return np.where(keep, x, 0.0) * factor(scale, p)


def embedding(weight, ids, padding_idx=None, **drop):
    weight, ids = np.asarray(weight, dtype=np.float64), np.asarray(ids).reshape(-1)
    valid = (ids >= 0) & (ids < weight.shape[0])
    if padding_idx is not None:
        valid &= ids != padding_idx
    rows = np.zeros((ids.size, weight.shape[1]))
    if weight.shape[0]:
        rows = dropped(weight[np.where(valid, ids, 0)], **drop)
    return np.where(valid[:, None], rows, 0.0)


def embedding_grad(ids, grads, num_rows, padding_idx=None, **drop):
    """(gradient, sum of the magnitudes of its terms, number of its terms by row)"""
    ids = np.asarray(ids).reshape(-1)
    rows = dropped(np.asarray(grads).reshape(ids.size, -1), **drop)
    valid = (ids >= 0) & (ids < num_rows)
    if padding_idx is not None:
        valid &= ids != padding_idx
    total, size = np.zeros((num_rows, rows.shape[1])), np.zeros((num_rows, rows.shape[1]))
    np.add.at(total, ids[valid], rows[valid])
    np.add.at(size, ids[valid], np.abs(rows[valid]))
    return total, size, np.bincount(ids[valid], minlength=num_rows)

"""Residual path in 64 bits (numpy): LayerNorm, dropout from the counter-based generator, residual add, and
their gradients, written from the formulas.  The keep mask is Philox4x32-10 (Salmon, Moraes, Dror, Shaw:
Parallel random numbers: as easy as 1, 2, 3, 2011): element e of the mask tensor takes word e % 4 of the block with
key = seed and counter = (e // 4, offset) and is dropped if it is below round(p * 2**32)."""

from __future__ import annotations

import numpy as np

LOW = 0xFFFFFFFF


def philox4x32(counter, key, rounds: int = 10):
    """One block: four 32-bit counter words and two key words (Python ints) -> four words."""
    c, k = list(counter), list(key)
    for _ in range(rounds):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k[0], q & LOW, (p >> 32) ^ c[3] ^ k[1], p & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return c


def words(count: int, seed: int, offset: int) -> np.ndarray:
    """The first `count` words of (seed, offset), uint32."""
    m = np.arange(-(-count // 4), dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    c = [m & low, m >> half, np.full_like(m, offset & LOW), np.full_like(m, offset >> 32)]
    k = [seed & LOW, seed >> 32]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return np.stack(c, 1).reshape(-1)[:count].astype(np.uint32)


def keep_mask(shape, p: float, seed: int, offset: int = 0, share=()) -> np.ndarray:
    """Boolean keep mask, size 1 along the axes in `share`."""
    shared = {a % len(shape) for a in share}
    mshape = [1 if a in shared else n for a, n in enumerate(shape)]
    w = words(int(np.prod(mshape, dtype=np.int64)), seed, offset).astype(np.uint64)
    return (w >= np.uint64(int(p * 2.0 ** 32 + 0.5))).reshape(mshape)


def scale_of(p: float) -> float:
    """1 / (1 - p) as the 32-bit number that kept values are multiplied by (0 for p = 1)."""
    return float(np.float32(1.0 / (1.0 - p))) if p < 1.0 else 0.0


def dropout_add_ref(z, y, p, seed, offset=0, share=()):
    """z + dropout(y) in float64 (z None: dropout(y))."""
    y = np.asarray(y, np.float64)
    keep = np.broadcast_to(keep_mask(y.shape, p, seed, offset, share), y.shape)
    with np.errstate(invalid="ignore"):
        d = np.where(keep, y * scale_of(p), 0.0)
    return d if z is None else np.asarray(z, np.float64) + d


def layer_norm_ref(x, w=None, b=None, eps=1e-5):
    """h, xh, rstd in float64."""
    x = np.asarray(x, np.float64)
    n = x.shape[-1]
    mean = x.sum(-1, keepdims=True) / n
    var = ((x - mean) ** 2).sum(-1, keepdims=True) / n
    rstd = 1.0 / np.sqrt(var + eps)
    xh = (x - mean) * rstd
    h = xh * (1.0 if w is None else np.asarray(w, np.float64)) + (0.0 if b is None else np.asarray(b, np.float64))
    return h, xh, rstd


def layer_norm_grad_ref(dh, xh, rstd, w=None):
    """(dx, dw, db) in float64."""
    dh = np.asarray(dh, np.float64)
    g = dh * (1.0 if w is None else np.asarray(w, np.float64))
    dx = rstd * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
    lead = tuple(range(dh.ndim - 1))
    return dx, (dh * xh).sum(lead), dh.sum(lead)

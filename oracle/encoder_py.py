"""The encoder operators from their definitions, in 64 bits: numpy, one formula each, nothing shared with the kernels.

Every function takes arrays of any float type and computes in float64.  Next to a result stands what bounds a kernel's
error: `size`, the sum of the magnitudes of what is added up for each value.
"""
from __future__ import annotations

import math

import numpy as np


def philox4x32(counter, key):
    """Philox4x32-10 of J. Salmon, M. Moraes, R. Dror and D. Shaw, "Parallel random numbers: as easy as 1, 2, 3" (2011);
    counter: four uint64 arrays of 32-bit words, key: two words."""
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    c = [np.asarray(w, u) for w in counter]
    k = [int(key[0]), int(key[1])]
    for _ in range(10):
        a, b = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(b >> u(32)) ^ c[1] ^ u(k[0]), b & low, (a >> u(32)) ^ c[3] ^ u(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return c


def multipliers(rows, cols, p, seed, offset, first_row=0):
    """What a dropout multiplies each value of a matrix by: 0 or the reciprocal of the share that is kept."""
    dropped = math.floor(p * 65536 + 0.5)
    if dropped == 0:
        return np.ones((rows, cols))
    row, block = np.meshgrid(np.arange(first_row, first_row + rows, dtype=np.uint64), np.arange((cols + 7) // 8, dtype=np.uint64), indexing="ij")
    words = philox4x32([block, row & np.uint64(0xFFFFFFFF), row >> np.uint64(32), np.full_like(row, offset)], (seed % 2**32, seed >> 32))
    halves = np.stack([half for w in words for half in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=2).reshape(rows, -1)[:, :cols]
    return np.where(halves >= dropped, 65536.0 / max(65536 - dropped, 1), 0.0)


def dropped(x, m):
    """x times the multipliers, and 0 where they are 0 whatever x is."""
    return np.where(m == 0, 0.0, np.asarray(x, np.float64) * np.where(m == 0, 1.0, m))


def places(offsets, count):
    """Of every token its place in its row, -1 for what belongs to none."""
    at = np.full(count, -1, np.int64)
    for first, last in zip(offsets[:-1], offsets[1:]):
        at[first:last] = np.arange(last - first)
    return at


def embedding(offsets, ids, table, positions=None):
    at, ids = places(offsets, len(ids)), np.asarray(ids, np.int64)
    known = (at >= 0) & (ids >= 0) & (ids < table.shape[0])
    out = np.zeros((len(ids), table.shape[1]))
    out[known] += table.astype(np.float64)[ids[known]]
    size = np.abs(out)
    if positions is not None:
        placed = (at >= 0) & (at < positions.shape[0])
        more = positions.astype(np.float64)[at[placed]]
        out[placed] += more
        size[placed] += np.abs(more)
    return out, size


def embedding_backward(offsets, ids, grad, vocabulary, count_places):
    at, ids, grad = places(offsets, len(ids)), np.asarray(ids, np.int64), grad.astype(np.float64)
    known = (at >= 0) & (ids >= 0) & (ids < vocabulary)
    placed = (at >= 0) & (at < count_places)
    result = []
    for values in (grad, np.abs(grad)):
        table, positions = np.zeros((vocabulary, grad.shape[1])), np.zeros((count_places, grad.shape[1]))
        np.add.at(table, ids[known], values[known])
        np.add.at(positions, at[placed], values[placed])
        result.append((table, positions))
    return result  # [(gradients), (sizes)]


def layer_norm(x, weight, bias, eps, residual=None, m=None):
    s = np.asarray(x, np.float64) if m is None else dropped(x, m)
    if residual is not None:
        s = s + residual.astype(np.float64)
    mean = s.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(np.square(s - mean).mean(1, keepdims=True) + eps)
    return (s - mean) * rstd * weight + bias, s, mean[:, 0], rstd[:, 0]


def layer_norm_backward(grad, s, mean, rstd, weight, sum_grad=None, m=None):
    grad, s, mean, rstd = (np.asarray(a, np.float64) for a in (grad, s, mean, rstd))
    h = (s - mean[:, None]) * rstd[:, None]
    a = grad * weight
    d = rstd[:, None] * (a - a.mean(1, keepdims=True) - h * (a * h).mean(1, keepdims=True))
    size = rstd[:, None] * (np.abs(a) + np.abs(a).mean(1, keepdims=True) + np.abs(h) * np.abs(a * h).mean(1, keepdims=True))
    if sum_grad is not None:
        d, size = d + sum_grad, size + np.abs(sum_grad)
    return d if m is None else dropped(d, m), d, (grad * h).sum(0), grad.sum(0), size, (np.abs(grad * h)).sum(0), np.abs(grad).sum(0)


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activate(z, name):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z**3)))
    if name == "silu":
        return z / (1 + np.exp(-z))
    return z


def slope(z, name):
    if name == "relu":
        return np.where(z > 0, 1.0, 0.0)
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = np.tanh(c * (z + 0.044715 * z**3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return s + z * s * (1 - s)
    return np.ones_like(z)


def linear(x, weight, bias=None, activation="none", residual=None):
    """(out, z, the size of z)."""
    x, weight = x.astype(np.float64), weight.astype(np.float64)
    z, size = x @ weight.T, np.abs(x) @ np.abs(weight).T
    if bias is not None:
        z, size = z + bias, size + np.abs(bias)
    out = activate(z, activation)
    return out if residual is None else out + residual, z, size


def linear_backward(grad, x, weight, activation="none", z=None):
    """((gradients of x, weight, bias), (their sizes))."""
    x, weight, d = x.astype(np.float64), weight.astype(np.float64), grad.astype(np.float64)
    if activation != "none":
        d = d * slope(z.astype(np.float64), activation)
    e = np.abs(d)
    return (d @ weight, d.T @ x, d.sum(0)), (e @ np.abs(weight), e.T @ np.abs(x), e.sum(0))

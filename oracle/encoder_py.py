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


def positions(offsets, count, starts=None):
    """Of every token its position, None for what belongs to no row."""
    at = [None] * count
    for r, (first, last) in enumerate(zip(offsets[:-1], offsets[1:])):
        for t in range(first, last):
            at[t] = int(t - first) + (int(starts[r]) if starts is not None else 0)
    return at


def rotary(x, offsets, frequencies, starts=None, layout="half", inverse=False, magnitude=1.0):
    """(out, of every value that was turned the sum of the magnitudes that it was made of, 0 for what is copied)."""
    x = np.asarray(x, np.float64)
    out, size, n = x.copy(), np.zeros(x.shape), len(frequencies)
    a, b = (slice(0, n), slice(n, 2 * n)) if layout == "half" else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    for t, at in enumerate(positions(offsets, len(x), starts)):
        if at is None:
            continue
        angle = np.asarray(at * np.asarray(frequencies, np.longdouble) * (-1 if inverse else 1))
        c, s = np.cos(angle).astype(np.float64) * magnitude, np.sin(angle).astype(np.float64) * magnitude
        p, q = x[t][:, a], x[t][:, b]
        out[t][:, a], out[t][:, b] = p * c - q * s, p * s + q * c
        size[t][:, a] = size[t][:, b] = (np.abs(p) + np.abs(q)) * abs(magnitude)
    return out, size


def _rows_seen(offsets, key_offsets, key_lengths, causal):
    """(the tokens, the keys, [tokens, keys] which of them see which) of every row."""
    for r in range(len(offsets) - 1):
        t = slice(int(offsets[r]), int(offsets[r + 1]))
        count = int(key_offsets[r + 1] - key_offsets[r])
        if key_lengths is not None:
            count = max(0, min(count, int(key_lengths[r])))
        u = slice(int(key_offsets[r]), int(key_offsets[r]) + count)
        i, j = np.arange(t.stop - t.start)[:, None], np.arange(count)[None, :]
        yield t, u, (j <= i + count - (t.stop - t.start)) if causal else np.ones((len(i), count), bool)


def attention(q, k, v, offsets, key_offsets=None, key_lengths=None, causal=False, scale=None, unit=0.0, tiny=0.0, eps=2.0**-24):
    """(out, logsum [heads, tokens], what a kernel's out may be off by before it is rounded, the same for logsum).  unit: by how much of itself
    an exponential may be off that is rounded before it is multiplied, tiny: by how much where it is smaller than its type's normal
    numbers (next to a sum of at least 1, that of the largest score); out is divided by the sum of what was rounded, which is off by as much of itself.  A score of `width` products held in 32 bits is off by
    eps a product and addition, in proportion to the magnitudes that it adds up, twice where they are cut off instead of
    rounded; its difference from the largest score or the logsum by eps of both; the exponential follows."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    key_offsets = offsets if key_offsets is None else key_offsets
    scale, each, width = q.shape[2] ** -0.5 if scale is None else scale, q.shape[1] // k.shape[1], q.shape[2]
    out, off = np.zeros(q.shape), np.zeros(q.shape)
    logsum, log_off = np.full(q.shape[:2][::-1], -np.inf), np.zeros(q.shape[:2][::-1])
    for t, u, sees in _rows_seen(offsets, key_offsets, key_lengths, causal):
        any_seen = sees.any(1)
        for h in range(q.shape[1]):
            for i in np.flatnonzero(any_seen):
                at, keys = t.start + i, np.flatnonzero(sees[i]) + u.start
                kk, vv = k[keys, h // each], v[keys, h // each]
                s = scale * (kk @ q[at, h])
                top = s.max()
                e = np.exp(s - top)
                logsum[h, at] = top + np.log(e.sum())
                p = e / e.sum()
                out[at, h] = p @ vv
                score_off = score_error(scale * (np.abs(kk) @ np.abs(q[at, h])), abs(top), width, eps)
                worst = score_off.max()
                off[at, h] = (p * (unit + score_off + worst + 2 * (len(keys) + 8) * eps) + tiny) @ np.abs(vv) + (unit + tiny * len(keys)) * np.abs(out[at, h])
                log_off[h, at] = worst + 2 * (len(keys) + 8) * eps
    return out, logsum, off, log_off


def score_error(size, top, width, eps):
    return eps * (2 * (width + 4) * size + 4 * top + 8)


def attention_backward(grad, q, k, v, out, logsum, offsets, key_offsets=None, key_lengths=None, causal=False, scale=None, unit=0.0, tiny=0.0, eps=2.0**-24):
    """((gradients of q, k, v), (what a kernel's may be off by before they are rounded)), from out and logsum as they are given."""
    grad, q, k, v, out, logsum = (np.asarray(x, np.float64) for x in (grad, q, k, v, out, logsum))
    key_offsets = offsets if key_offsets is None else key_offsets
    scale, each, width = q.shape[2] ** -0.5 if scale is None else scale, q.shape[1] // k.shape[1], q.shape[2]
    results, offs = [np.zeros(x.shape) for x in (q, k, v)], [np.zeros(x.shape) for x in (q, k, v)]
    for t, u, sees in _rows_seen(offsets, key_offsets, key_lengths, causal):
        if not sees.any():
            continue
        for h in range(q.shape[1]):
            qh, gh, oh, kh, vh = q[t, h], grad[t, h], out[t, h], k[u, h // each], v[u, h // each]
            log = np.where(sees.any(1), logsum[h, t], 0.0)[:, None]
            s = scale * (qh @ kh.T)
            p = np.where(sees, np.exp(np.where(sees, s - log, 0.0)), 0.0)
            dp, delta = gh @ vh.T, (gh * oh).sum(1)[:, None]
            ds = p * (dp - delta)
            e = score_error(scale * (np.abs(qh) @ np.abs(kh).T), np.abs(log), width, eps) + 8 * eps
            dp_off = 2 * (width + 4) * eps * (np.abs(gh) @ np.abs(vh).T + (np.abs(gh) * np.abs(oh)).sum(1)[:, None])
            ds_off = 1.1 * (np.abs(ds) * (unit + e) + p * dp_off) + np.where(sees, tiny, 0.0)
            longest = 2 * (max(s.shape) * each + 8) * eps
            results[0][t, h] = scale * (ds @ kh)
            offs[0][t, h] = scale * ((ds_off + longest * np.abs(ds)) @ np.abs(kh))
            results[1][u, h // each] += scale * (ds.T @ qh)
            offs[1][u, h // each] += scale * ((ds_off + longest * np.abs(ds)).T @ np.abs(qh))
            results[2][u, h // each] += p.T @ gh
            offs[2][u, h // each] += (1.1 * p * (unit + e + longest) + np.where(sees, tiny, 0.0)).T @ np.abs(gh)
    return results, offs

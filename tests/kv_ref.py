"""Plain 64-bit restatement of the KV-cache operators (include/brrr.h), entry by entry and row by row, on numpy arrays.

Caches are [seq][kv head][slot][dim] arrays of the values that the stored type holds."""
import math

import numpy as np


def depth(mask, i):
    return bin(mask & ~(1 << i)).count("1")


def chain(rows):
    return [(1 << (i + 1)) - 1 for i in range(rows)]


def sees(masks, count, length, window, i, t):
    """masks: of one entry, any bits; whether row i sees slot t."""
    live = (1 << count) - 1
    di = depth(masks[i] & live, i)
    if t < length:
        return window == 0 or t >= length + di + 1 - window
    j = t - length
    if j >= count or not masks[i] >> j & 1:
        return False
    return window == 0 or di - depth(masks[j] & live, j) < window


def attend(q, k, v, slots, scale, sink=None):
    """One query head over the given slots: (out, lse, weights)."""
    s = (k[slots] @ q) * scale if len(slots) else np.zeros(0)
    top = max([*s.tolist(), *([] if sink is None else [sink])], default=-math.inf)
    if top == -math.inf:
        return np.zeros(v.shape[1]), -math.inf, np.zeros(0)
    p = np.exp(s - top)
    total = p.sum() + (0.0 if sink is None else math.exp(sink - top))
    return (p / total) @ v[slots] if len(slots) else np.zeros(v.shape[1]), top + math.log(total), p / total


def tree(q, k, v, seq, length, count, masks, scale, window=0, sinks=None):
    """q [n][rows][heads][dim] -> out (zeros where no row is), lse, and [(b, i, h, slots, weights)]"""
    n, rows, heads, dim = q.shape
    per = heads // k.shape[1]
    out, lse, weights = np.zeros(q.shape), np.zeros(q.shape[:3]), []
    for b in range(n):
        for i in range(count[b]):
            slots = [t for t in range(length[b] + count[b]) if sees(masks[b], count[b], length[b], window, i, t)]
            for h in range(heads):
                out[b, i, h], lse[b, i, h], w = attend(q[b, i, h], k[seq[b], h // per], v[seq[b], h // per], slots, scale, None if sinks is None else sinks[h])
                weights.append((b, i, h, slots, w))
    return out, lse, weights


def rotate(x, rope):
    """x [heads][dim], rope [dim / 2][2]; single precision, each product and sum rounded."""
    half = x.shape[1] // 2
    a, b, c, s = x[:, :half], x[:, half:], rope[:, 0], rope[:, 1]
    return np.concatenate([a * c - b * s, a * s + b * c], 1)


def evict(weight, pos, keep, first, recent, end):
    """weight, pos: one head's entries -> the slot that each of the kept entries comes from."""
    n = len(weight)
    m = min(n, keep)
    w = np.where(np.isnan(weight), -np.inf, weight)
    order = sorted(range(n), key=lambda t: (not (pos[t] < first or (recent > 0 and pos[t] >= end - recent)), bool(np.isnan(weight[t])), -w[t], t))
    kept = set(order[:m])
    spare = sorted(t for t in kept if t >= m)
    return [t if t in kept else spare.pop(0) for t in range(m)]


def choose(q, means, length, block, nsel, first, local):
    """q [g][dim] float32, means [blocks][dim] float32 -> the blocks of one kv head in ascending order"""
    nb = -(-length // block)
    if nb <= nsel:
        return list(range(nb))
    must = [j for j in range(nb) if j < first or j >= nb - local]
    score = (q.astype(np.float64) @ means[: nb].astype(np.float64).T).max(0).astype(np.float32) if len(means) else np.zeros(0)
    free = sorted((j for j in range(nb) if j not in set(must)), key=lambda j: (bool(np.isnan(score[j])), -score[j] if not np.isnan(score[j]) else 0.0, j))
    return sorted(must + free[: nsel - len(must)])

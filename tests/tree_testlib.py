"""Attention of trees of drafts in 64 bits: what each node sees, and O with the bound of ``paged_testlib`` (the same
kernels' rounding)."""

import random

import numpy as np


def shape(kind, n, seed=0):
    """Parents of n nodes: 'chain', 'star', 'roots', 'level' (two or three children each), 'any' (any node before, some
    roots), 'odd' (numbers that are no node before, too)."""
    rng = random.Random(seed)
    if kind == "chain":
        return list(range(-1, n - 1))
    if kind == "star":
        return [-1] + [0] * (n - 1) if n else []
    if kind == "roots":
        return [-1] * n
    if kind == "level":
        return [-1 if i == 0 else (i - 1) // rng.choice((2, 3)) for i in range(n)]
    if kind == "any":
        return [rng.randint(-1, i - 1) if rng.random() < 0.3 else max(-1, i - rng.randint(1, 4)) for i in range(n)]
    odd = (-7, 2 ** 31 - 1, -2 ** 31, n + 5)
    return [rng.choice(odd + (i, i + 1)) if rng.random() < 0.1 else max(-1, i - rng.randint(1, 9)) for i in range(n)]


def seen_by(parents, base, length, window=None, sinks=0):
    """Truth values [n, length] of what the nodes see of a sequence's keys (its last ones, from base on, are theirs)."""
    n = len(parents)
    above, depth = [], []
    for i, p in enumerate(parents):
        up = above[p] if 0 <= p < i else []
        above.append(up + [i])
        depth.append(len(up))
    seen = np.zeros((n, length), dtype=bool)
    for i in range(n):
        pos = base + depth[i]
        for j in range(min(base, length)):
            seen[i, j] = not window or pos - j < window or j < sinks
        for a in above[i]:
            if 0 <= base + a < length:
                seen[i, base + a] = not window or depth[i] - depth[a] < window or base + depth[a] < sinks
    return seen


def attend_seen(q, k, v, seen, scale=None):
    """q [n, Hq, D], k / v [L, H, D], seen [n, L] -> (O, bound) in 64 bits; only what is seen is touched."""
    q, k, v = (np.asarray(x.detach().cpu().double()) for x in (q, k, v))
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = dim ** -0.5 if scale is None else scale
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for i in range(n):
        if not seen[i].any():
            continue
        ks, vs = k[seen[i]], v[seen[i]]
        for h in range(k.shape[1]):
            rows = slice(h * group, (h + 1) * group)
            with np.errstate(invalid="ignore", over="ignore"):
                s = q[i, rows] @ ks[:, h].T * scale
                p = np.exp(s - s.max(1, keepdims=True))
                p /= p.sum(1, keepdims=True)
                o, a = p @ vs[:, h], p @ np.abs(vs[:, h])
                most = (np.abs(q[i, rows]) @ np.abs(ks[:, h]).T).max() * scale
            out[i, rows] = o
            bound[i, rows] = (2 ** -8 * np.abs(o) + (2 ** -8 + 2 ** -12 + 2 * (dim + 2) * 2 ** -24 * most) * a
                              + 2.0 ** -126 * (1 + np.abs(vs[:, h]).sum(0)))
    return out, bound

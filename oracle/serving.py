"""64-bit restatements of the serving operators (attention over a shared prefix, eviction from
the cache, logits processing), row by row and head by head. The reference has none of them
(orchard/model.py:112-144,244-252: attention per sequence, every position kept, plain logits)."""

from __future__ import annotations

import numpy as np


def attention_prefix(q, prefix_k, prefix_v, units, k_cache, v_cache, lens, slots, mass=None):
    """q [M, nh, hd]; prefix_k/v [prefixes, nkv, cap, hd]; units rows of (row0, rows, prefix,
    length); caches [slots, nkv, max_seq, hd]. Returns (out, weighted |v|, new mass, largest
    sum of |q k|): the second and the last are what error bounds are made of."""
    M, nh, hd = q.shape
    nkv = k_cache.shape[1]
    G = nh // nkv
    out = np.zeros((M, nh, hd))
    absv = np.zeros((M, nh, hd))
    mass = None if mass is None else mass.astype(np.float64).copy()
    big = 0.0
    for m in range(M):
        L, t = int(lens[m]), int(slots[m])
        own = [u for u in units if u[0] <= m < u[0] + u[1]]
        for h in range(nh):
            kv = h // G
            k, v = k_cache[t, kv, :L].astype(np.float64), v_cache[t, kv, :L].astype(np.float64)
            if own:
                _, _, p, n = own[0]
                k = np.concatenate([prefix_k[p, kv, :n].astype(np.float64), k])
                v = np.concatenate([prefix_v[p, kv, :n].astype(np.float64), v])
            if len(k) == 0:
                continue
            x = q[m, h].astype(np.float64)
            s = k @ x / np.sqrt(hd)
            big = max(big, float((np.abs(k) @ np.abs(x)).max() / np.sqrt(hd)))
            e = np.exp(s - s.max())
            e /= e.sum()
            out[m, h], absv[m, h] = e @ v, e @ np.abs(v)
            if mass is not None and L:
                w = e[len(e) - L:]
                mass[t, kv, :L - 1] += w[:-1]
                # the newest entry starts from its weight; later heads of the group add to it
                mass[t, kv, L - 1] = w[-1] + (mass[t, kv, L - 1] if h % G else 0.0)
    return out, absv, mass, big


def cache_evict(mass, positions, length, budget, recent):
    """One (row, K/V head): for each of the min(length, budget) entries left, the index it had."""
    n = min(length, budget)
    m, p = mass[:length].astype(np.float64), positions[:length].astype(np.int64)
    if n == 0:
        return np.zeros(0, np.int64)
    m = np.where(np.isnan(m), -np.inf, m)
    low = np.isnan(mass[:length].astype(np.float64))  # below -inf
    guard = p > p.max() - recent
    order = sorted(range(length), key=lambda e: (not guard[e], low[e], -m[e], e))
    kept = np.zeros(length, bool)
    kept[order[:n]] = True
    src = np.arange(n)
    src[~kept[:n]] = np.flatnonzero(kept[n:]) + n
    return src


def logits_process(row, base=0, history=(), gen_start=0, penalties=None, bias=(), allowed=None):
    """One row of logits; bias: (id, value) pairs; allowed: None or the set of allowed ids."""
    x = row.astype(np.float64).copy()
    V = len(x)
    if penalties is not None:
        rep, pres, freq = (float(v) for v in penalties)
        for v in set(int(t) for t in history):
            i = v - base
            if 0 <= i < V:
                x[i] = x[i] / rep if x[i] > 0 else x[i] * rep
                c = sum(1 for t in history[gen_start:] if int(t) == v)
                if c:
                    x[i] -= freq * c + pres
    for v, b in dict((int(v), float(b)) for v, b in bias).items():
        if 0 <= v - base < V:
            x[v - base] += b
    if allowed is not None:
        for i in range(V):
            if base + i not in allowed:
                x[i] = -np.inf
    return x

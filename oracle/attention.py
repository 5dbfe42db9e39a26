"""Attention and cache eviction in 64 bits (test infrastructure).

Written from the formulas: s_j = scale q.k_j, w = softmax(s), out = sum_j w_j v_j,
lse = log sum_j exp(s_j).  Besides the results each function gives what error
bounds need: ``spread`` = sum_j w_j |v_j| (a relative error e of every weight
moves the output by at most e * spread) and ``mag`` = max_j scale sum_d |q_d k_jd|
(an error of the products' sums is relative to it).
"""
from __future__ import annotations

import numpy as np


def attend(q, k, v, scale, causal=False):
    """q [n, Hq, D], k, v [L, Hkv, D] (float64) -> dict of out [n, Hq, D], lse [n, Hq],
    spread [n, Hq, D], mag [n, Hq], weight [Hkv, L] (weights summed over rows and query heads)."""
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    G = Hq // Hkv
    out, spread = np.zeros((n, Hq, D)), np.zeros((n, Hq, D))
    lse, mag, weight = np.full((n, Hq), -np.inf), np.zeros((n, Hq)), np.zeros((Hkv, L))
    for i in range(n):
        m = max(0, i + L - n + 1) if causal else L
        if m == 0:
            continue
        for h in range(Hkv):
            qs = q[i, h * G:(h + 1) * G]
            s = scale * qs @ k[:m, h].T
            top = s.max(1, keepdims=True)
            e = np.exp(s - top)
            w = e / e.sum(1, keepdims=True)
            sl = slice(h * G, (h + 1) * G)
            out[i, sl] = w @ v[:m, h]
            spread[i, sl] = w @ np.abs(v[:m, h])
            lse[i, sl] = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
            mag[i, sl] = (scale * np.abs(qs) @ np.abs(k[:m, h]).T).max(1)
            weight[h, :m] += w.sum(0)
    return dict(out=out, lse=lse, spread=spread, mag=mag, weight=weight)


def evict(mass, positions, length, seen, budget, recent, sinks):
    """One head of one sequence: (holes, tails), the entries filled and the entries they take, in order."""
    if length <= budget:
        return [], []
    key = []
    for i in range(length):
        p = positions[i]
        guarded = p >= seen - recent or p < sinks
        key.append((0 if guarded else 1, 0.0 if guarded else -float(mass[i]), i))
    kept = sorted(k[2] for k in sorted(key)[:budget])
    inside = set(kept)
    return [i for i in range(budget) if i not in inside], [i for i in kept if i >= budget]

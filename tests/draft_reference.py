"""The drafted-decoding operators in float64 numpy, from their definitions."""

import numpy as np


def ancestors(parents, i):
    """Nodes that node i sees, itself among them; empty where i is padding."""
    got = []
    while True:
        if not -1 <= parents[i] < i:
            return []
        got.append(i)
        if parents[i] == -1:
            return sorted(got)
        i = parents[i]


def attention(q, k_cache, v_cache, lens, k_new, v_new, parents, scale):
    """Returns out, lse, and for bounds on the error sum_k p_k |v_k|, the
    largest sum |q_d k_d| scale and the largest number of keys of each row."""
    B, n, Hq, D = q.shape
    G = Hq // k_cache.shape[1]
    out, mag = np.zeros((B, n, Hq, D)), np.zeros((B, n, Hq, D))
    lse, big = np.full((B, n, Hq), -np.inf), np.zeros((B, n, Hq))
    keys = np.zeros((B, n, Hq), int)
    for b in range(B):
        m = min(max(int(lens[b]), 0), k_cache.shape[2])
        for i in range(n):
            see = ancestors(list(parents[b]), i)
            if not see:
                continue
            for h in range(Hq):
                k = np.concatenate([k_cache[b, h // G, :m], k_new[b, see, h // G]])
                v = np.concatenate([v_cache[b, h // G, :m], v_new[b, see, h // G]])
                s = k @ q[b, i, h] * scale
                top = s.max()
                e = np.exp(s - top)
                p = e / e.sum()
                lse[b, i, h] = top + np.log(e.sum())
                with np.errstate(invalid="ignore"):
                    out[b, i, h] = p @ v
                mag[b, i, h] = p @ np.abs(v)
                big[b, i, h] = (np.abs(k) @ np.abs(q[b, i, h])).max() * abs(scale)
                keys[b, i, h] = len(s)
    return out, lse, mag, big, keys


def verify(target, draft, tokens, parents, uniforms):
    B, n = tokens.shape
    V = target.shape[2]
    path, count, token = np.full((B, n), -1), np.zeros(B, int), np.zeros(B, int)
    for b in range(B):
        at, go = -1, True
        p = np.where(target[b, 0] > 0, target[b, 0], 0.0)
        q = np.where(draft[b, 0] > 0, draft[b, 0], 0.0)
        while go:
            go = False
            for c in range(at + 1, n):
                if parents[b, c] != at:
                    continue
                x = tokens[b, c]
                if 0 <= x < V and uniforms[b, c] * q[x] < p[x]:
                    path[b, count[b]] = c
                    count[b] += 1
                    at, go = c, True
                    p = np.where(target[b, c + 1] > 0, target[b, c + 1], 0.0)
                    q = np.where(draft[b, c + 1] > 0, draft[b, c + 1], 0.0)
                    break
                rest = np.maximum(p - q, 0.0)
                if rest.sum() > 0:
                    p = rest / rest.sum()
        cdf = np.cumsum(p)
        over = np.nonzero(cdf > uniforms[b, n] * cdf[-1])[0]
        some = np.nonzero(p > 0)[0]
        token[b] = over[0] if len(over) else some[-1] if len(some) else 0
    return path, count, token


def fits(path, count, length, n, cap):
    return 0 <= count <= n and 0 <= length and length + count <= cap and all(0 <= x < n for x in path[:count])


def accumulate(q, lse, k_cache, lens, path, count, acc, scale):
    B, n, Hq, _ = q.shape
    Hk = k_cache.shape[1]
    acc = acc.copy()
    for b in range(B):
        m, a = int(lens[b]), int(count[b])
        if not fits(path[b], a, m, n, k_cache.shape[2]):
            continue
        acc[b, :, m:m + a] = 0.0
        for j in range(a):
            node = path[b, j]
            for h in range(Hq):
                g = h // (Hq // Hk)
                s = k_cache[b, g, :m + j + 1] @ q[b, node, h] * scale
                acc[b, g, :m + j + 1] += np.exp(s - lse[b, node, h])
    return acc


def keep(acc, length, budget, recent):
    """The rows that stay, in order."""
    if length <= budget:
        return np.arange(length)
    w = np.where(np.isnan(acc[:length - recent]), -np.inf, acc[:length - recent])
    order = sorted(range(length - recent), key=lambda i: (-w[i], i))[:budget - recent]
    # a weight that is not a number stays behind those of -inf
    nan = np.isnan(acc[:length - recent])
    if nan.any():
        order = sorted(range(length - recent), key=lambda i: (nan[i], -w[i], i))[:budget - recent]
    return np.concatenate([np.sort(np.array(order, int)), np.arange(length - recent, length)])

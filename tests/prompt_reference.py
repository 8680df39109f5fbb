"""Packed prompts and 4-bit cache rows in float64 numpy, from their
definitions."""

import numpy as np

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# every scale that a row may have: byte b is (1 + m / 8) 2^(e - 15), or m / 8 2^-14 where e = 0
SCALES = np.array([b * 2.0 ** -17 if b < 8 else (1 + b % 8 / 8) * 2.0 ** (b // 8 - 15) for b in range(0xE3)])


def starts_of(starts, tokens):
    return np.maximum.accumulate(np.clip(np.asarray(starts, np.int64), 0, tokens))


def prompt(q, k, v, starts, scale):
    """out and lse, and for bounds on the error sum_j p_j |v_j|, the largest
    sum |q_d k_d| scale and the number of keys of each row."""
    T, Hq, D = q.shape
    G = Hq // k.shape[1]
    out, mag = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    lse, big, keys = np.full((T, Hq), -np.inf), np.zeros((T, Hq)), np.zeros((T, Hq), int)
    s = starts_of(starts, T)
    for a, e in zip(s, s[1:]):
        if a == e:
            continue
        n = e - a
        hidden = ~np.tri(n, dtype=bool)
        for h in range(Hq):
            kk, vv = k[a:e, h // G], v[a:e, h // G]
            x = np.where(hidden, -np.inf, q[a:e, h] @ kk.T * scale)
            top = x.max(1, keepdims=True)
            p = np.exp(x - top)
            total = p.sum(1, keepdims=True)
            p /= total
            lse[a:e, h] = (top + np.log(total))[:, 0]
            out[a:e, h], mag[a:e, h] = p @ vv, p @ np.abs(vv)
            big[a:e, h] = np.where(hidden, 0.0, np.abs(q[a:e, h]) @ np.abs(kk).T).max(1) * abs(scale)
            keys[a:e, h] = np.arange(1, n + 1)
    return out, lse, mag, big, keys


def row_bytes(D):
    g = -(-D // 16)
    return -(-9 * g // 4) * 4


def nearest(x, table):
    """Index of the nearest entry of a rising table, the even one in the middle."""
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    a, b = x - table[hi - 1], table[hi] - x
    return np.where((b < a) | ((a == b) & (hi % 2 == 0)), hi, hi - 1)


def pack(x):
    """Rows [..., row_bytes(D)] of the values x [..., D]."""
    D = x.shape[-1]
    g = -(-D // 16)
    x = np.concatenate([np.asarray(x, np.float64), np.zeros((*x.shape[:-1], 16 * g - D))], -1)
    x = x.reshape(*x.shape[:-1], g, 16)
    fine = np.isfinite(x).all(-1)
    y = np.where(fine[..., None], x, 0.0)
    b = nearest(np.abs(y).max(-1) / 6, SCALES)
    s = SCALES[b]
    code = np.where((s > 0)[..., None], nearest(np.abs(y) / np.where(s > 0, s, 1.0)[..., None], VALUES), 0)
    code = np.where(fine[..., None], code + 8 * np.signbit(x), 0).astype(np.uint8).reshape(*x.shape[:-2], 16 * g)
    scale = np.where(fine, b, 0xFC).astype(np.uint8)
    rest = np.zeros((*scale.shape[:-1], row_bytes(D) - 9 * g), np.uint8)
    return np.concatenate([code[..., 0::2] + 16 * code[..., 1::2], scale, rest], -1)


def unpack(rows, D):
    """The values of rows, [..., D]; NaN where a group holds none."""
    g = -(-D // 16)
    code = np.stack([rows[..., :8 * g] & 15, rows[..., :8 * g] >> 4], -1).reshape(*rows.shape[:-1], g, 16)
    b = rows[..., 8 * g:9 * g]
    s = np.where(b < len(SCALES), SCALES[np.minimum(b, len(SCALES) - 1)], np.nan)
    x = np.where(code & 8, -1.0, 1.0) * VALUES[code & 7] * s[..., None]
    return x.reshape(*rows.shape[:-1], 16 * g)[..., :D]


def fill(cache, lens, rows, starts):
    """The cache [B, H, capacity, ...] and the lengths after the packed rows
    [T, H, ...] are appended."""
    cache, new = cache.copy(), np.array(lens)
    s = starts_of(starts, rows.shape[0])
    for b, (a, e) in enumerate(zip(s, s[1:])):
        m = int(lens[b])
        if 0 <= m and m + e - a <= cache.shape[2]:
            cache[b, :, m:m + e - a] = np.moveaxis(rows[a:e], 0, 1)
            new[b] = m + e - a
    return cache, new

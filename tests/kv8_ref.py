"""Plain 64-bit forms of the 8-bit KV cache operators, for the tests."""
import numpy as np


def quantize(x):
    """x [..., hd] fp32 -> (codes int8, scales fp32): scale = max|x| * (1 / 127) in fp32, codes rounded half to
    even."""
    x = np.asarray(x, np.float32)
    peak = np.abs(x).max(-1)
    bad = ~np.isfinite(peak)
    scale = np.where(bad, 0, peak).astype(np.float32) * np.float32(1 / 127)
    s = np.where(scale > 0, scale, 1).astype(np.float64)[..., None]
    q = np.rint(np.where(bad[..., None], 0, x).astype(np.float64) / s)
    codes = np.where((scale > 0)[..., None], np.clip(q, -127, 127), 0).astype(np.int8)
    return codes, np.where(bad, np.float32(np.nan), scale)


def weight(x):
    """The framework's softmax weight of x = score - maximum <= 0."""
    x = np.where(x < -87.3, -87.3, x)
    return (12 + 6 * x + x * x) / (12 - 6 * x + x * x)


def attend(q, k, v):
    """q [G, hd], k / v [n, hd], one kv head.  Returns (out, tol): tol bounds the error of an fp32
    computation of out, element by element.

    A score formed with the error of 8 roundings of its absolute sum a = sum|q||k| / sqrt(hd) is off by at
    most d = 8 * 2^-24 * a, and so is the maximum.  |w'/w| <= 1 for x <= 0, so a weight is off by 2 d
    relative (8 more roundings for the quotient); numerator and denominator each by that, and by the
    roundings of their sums: at most 64 + n / 64 in a chain, since every kernel sums in blocks.  The two
    errors at most add up, times sum(w |v|) / sum(w).

    The products w * v_scale are held in fixed point, a half step of 2^-24 times the largest scale away at
    most: 2^-24 * max(scale) * sum|code| / sum(w) more.  (A key's scale is max|v| / 127.  The key with the
    largest scale has w >= 0.07 and is itself up to half a scale off its unquantised value, so this stays
    far below what the 8 bits cost.)"""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    n, hd = k.shape
    if n == 0:
        return np.zeros_like(q), np.zeros_like(q)
    z = q @ k.T / np.sqrt(hd)
    w = weight(z - z.max(1, keepdims=True))
    total = w.sum(1, keepdims=True)
    a = (np.abs(q) @ np.abs(k).T / np.sqrt(hd)).max(1, keepdims=True)
    d = 8 * 2.0 ** -24 * a
    rel = 2 * (2 * d + (8 + 64 + n / 64) * 2.0 ** -24)
    scale = np.abs(v).max(1, keepdims=True) / 127
    codes = np.abs(v) / np.where(scale > 0, scale, 1)
    return w @ v / total, rel * (w @ np.abs(v) / total) + 2.0 ** -24 * scale.max() * codes.sum(0) / total


def attend_rows(q, n_kv, keys):
    """q [B, n_heads, hd]; keys[b] = list of segments (arrays, slot, n) in key order, with arrays = (k codes,
    k scales, v codes, v scales), or None for a row that is left alone.  Returns (out, tol) as attend does."""
    B, n_heads, hd = q.shape
    group = n_heads // n_kv
    out, tol = np.zeros((2, B, n_heads, hd))
    for b in range(B):
        if keys[b] is None:
            out[b] = np.nan
            continue
        for g in range(n_kv):
            parts = [[c[0][s, g, :n].astype(np.float64) * c[1][s, g, :n, None].astype(np.float64),
                      c[2][s, g, :n].astype(np.float64) * c[3][s, g, :n, None].astype(np.float64)]
                     for c, s, n in keys[b]]
            k = np.concatenate([p[0] for p in parts])
            v = np.concatenate([p[1] for p in parts])
            h = slice(g * group, (g + 1) * group)
            out[b, h], tol[b, h] = attend(q[b, h], k, v)
    return out, tol

"""Plain models in float64 of attention with a sliding window and of the 4-bit rows."""
import math

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def sees(positions, keys, window, sinks):
    """[T, N] bool: position i sees key j if j <= i and (i - j < window or j < sinks)."""
    back = np.asarray(positions)[:, None] - np.arange(keys)[None, :]
    return (back >= 0) & ((back < window) | (np.arange(keys) < sinks)[None, :])


def forward(q, k, v, window, sinks, scale):
    """q [Hq, S, D], k, v [Hkv, S, D] of one batch element: O, LSE [Hq, S], and for bounds sum p |v| and the
    largest scale * sum |q k| of the keys that a row sees."""
    hq, s, _ = q.shape
    group = hq // k.shape[0]
    see = sees(np.arange(s), s, window, sinks)
    o, av, lse, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((hq, s)), np.zeros((hq, s))
    for h in range(hq):
        kk, vv = k[h // group], v[h // group]
        z = np.where(see, scale * (q[h] @ kk.T), -np.inf)
        m = z.max(1, keepdims=True)
        p = np.exp(z - m)
        l = p.sum(1, keepdims=True)
        o[h], av[h] = p @ vv / l, p @ np.abs(vv) / l
        lse[h] = (m + np.log(l))[:, 0]
        size[h] = np.where(see, scale * (np.abs(q[h]) @ np.abs(kk).T), 0).max(1)
    return o, lse, av, size


def backward(q, k, v, dout, o, lse, window, sinks, scale, h):
    """Gradients of one batch element from the forward's O and LSE, and how far each may be off when the
    products are sums in f32 of exact products, P and dS are rounded by h (half a step relative to the
    value), and so is the result."""
    hq, s, d = q.shape
    group = hq // k.shape[0]
    see = sees(np.arange(s), s, window, sinks)
    grads = [np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)]
    off = [np.zeros(x.shape) for x in grads]
    sums = (d + 16) * 2.0 ** -24
    for i in range(hq):
        g = i // group
        z = np.where(see, scale * (q[i] @ k[g].T), -np.inf)
        p = np.where(see, np.exp(z - lse[i][:, None]), 0)
        # of P, relative: the score's products, its scaling and LSE's (three roundings of their sizes), exp2
        size = np.where(see, scale * (np.abs(q[i]) @ np.abs(k[g]).T), 0)
        ep = size * sums + 2.0 ** -22 * (size + np.abs(lse[i][:, None])) + 2.0 ** -21
        dp = dout[i] @ v[g].T
        delta = (dout[i] * o[i]).sum(1)[:, None]
        ed = sums * (np.abs(dout[i]) @ np.abs(v[g]).T + (np.abs(dout[i] * o[i])).sum(1)[:, None])
        ds = p * (dp - delta)
        es = np.abs(ds) * (ep + h) + p * ed * (1 + ep + h) + 2.0 ** -22 * np.abs(ds)
        grads[0][i] += scale * ds @ k[g]
        grads[1][g] += scale * ds.T @ q[i]
        grads[2][g] += p.T @ dout[i]
        acc = s * group * 2.0 ** -24
        off[0][i] += scale * (es + acc * np.abs(ds)) @ np.abs(k[g])
        off[1][g] += scale * (es + acc * np.abs(ds)).T @ np.abs(q[i])
        off[2][g] += (p * (ep + h + acc)).T @ np.abs(dout[i])
    return grads, [e * (1 + h) + (h + 2.0 ** -22) * np.abs(x) for x, e in zip(grads, off)]


def to_rows(x):
    """The 4-bit rows (uint8 [n, row bytes]) of x [n, heads, dim] float64, f32 numbers."""
    n = x.shape[0]
    y = x.reshape(n, -1, 32)
    top = np.abs(y).max(2)
    bad = ~np.isfinite(y).all(2)
    with np.errstate(all="ignore"):
        e = np.ceil(np.log2(np.where(bad | (top == 0), 1.0, top) / 7.0))
        e = np.where(top >= 7.0 * np.exp2(e), e + 1, np.where(top < 7.0 * np.exp2(e - 1), e - 1, e))
        e = np.where(top == 0, -127, np.clip(e, -127, 125))
        a = np.abs(y) / np.exp2(e)[:, :, None]
    # ties to the even code
    edges = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]
    code = sum(((a >= x) if up else (a > x)).astype(np.uint8) for x, up in edges)
    code = np.where(bad[:, :, None], 0, code | (np.signbit(y).astype(np.uint8) << 3)).reshape(n, -1, 2)
    codes = code[:, :, 0] | (code[:, :, 1] << 4)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    row = np.concatenate([codes.astype(np.uint8), scales], 1)
    return np.pad(row, ((0, 0), (0, -row.shape[1] % 16)))


def from_rows(rows, heads, dim):
    """What 4-bit rows stand for, float64 [n, heads, dim]."""
    n, half = rows.shape[0], heads * dim // 2
    code = np.stack([rows[:, :half] & 15, rows[:, :half] >> 4], -1).reshape(n, -1, 32)
    scale = rows[:, half:half + heads * dim // 32].astype(np.float64)
    scale = np.where(scale == 255, np.nan, np.exp2(scale - 127))
    return (np.where(code & 8, -1.0, 1.0) * LEVELS[code & 7] * scale[:, :, None]).reshape(n, heads, dim)


def resolved(dim):
    return float(np.float32(1) / np.float32(math.sqrt(dim)))

"""Plain models of the device-resident batch's operators in Python integers and float64."""
import numpy as np


def reserve(table, ctx, new, mapped, free, count, max_new, page, pages):
    """The state after a reservation; arrays are copied."""
    table, ctx, mapped, free = (np.array(x) for x in (table, ctx, mapped, free))
    n, width = table.shape
    slots, granted = np.full((n, max_new), -1, np.int64), np.zeros(n, np.int64)
    top = int(count)
    kept = np.clip(mapped, 0, width)
    out = kept.copy()
    for s in range(n):
        if new[s] < 0:
            for j in range(kept[s]):
                if top < free.size:
                    free[top] = table[s, j]
                top += 1
            out[s] = 0
    top = min(top, free.size)
    wanted = taken = 0
    for s in range(n):
        if new[s] < 0:
            ctx[s] = 0
            continue
        total = int(ctx[s]) + int(new[s])
        if ctx[s] < 0 or new[s] == 0 or new[s] > max_new or total > width * page:
            continue
        need = max(0, -(-total // page) - int(kept[s]))
        wanted += need
        if need and wanted > top:
            continue
        for j in range(need):
            table[s, kept[s] + j] = free[top - 1 - taken - j]
        taken += need
        out[s] = kept[s] + need
        granted[s] = new[s]
        for t in range(int(new[s])):
            row = int(table[s, (ctx[s] + t) // page])
            if 0 <= row < pages:
                slots[s, t] = row * page + (ctx[s] + t) % page
    return {"table": table, "ctx": ctx, "mapped": out, "free": free, "count": top - taken,
            "granted": granted, "slots": slots}


def tree(parents, lens, ctx, max_tokens):
    """(seen [n, max_tokens, max_tokens] bool, positions) of drafted trees."""
    n = len(lens)
    seen = np.zeros((n, max_tokens, max_tokens), bool)
    positions = np.full((n, max_tokens), -1, np.int64)
    for s in range(n):
        if not 0 <= lens[s] <= max_tokens or ctx[s] < 0:
            continue
        for t in range(lens[s]):
            p = int(parents[s, t])
            if p < -1 or p >= t or (p >= 0 and not seen[s, p, p]):
                continue
            if p >= 0:
                seen[s, t] = seen[s, p]
            seen[s, t, t] = True
            positions[s, t] = ctx[s] + seen[s, t].sum() - 1
    return seen, positions


def pack(seen):
    """Bit masks [n, tokens, words] uint64 of seen [n, tokens, tokens]."""
    n, tokens, _ = seen.shape
    words = (tokens + 63) // 64
    bits = np.zeros((n, tokens, words * 64), np.uint64)
    bits[:, :, :tokens] = seen
    return (bits.reshape(n, tokens, words, 64) << np.arange(64, dtype=np.uint64)).sum(
        -1, dtype=np.uint64)


def angles(positions, dim, theta):
    """Angles [..., dim / 2]: f32 frequencies times f32 positions, rounded to f32, by definition."""
    freq = np.array([np.float32(theta) ** (np.float32(-2.0) * np.float32(j) / np.float32(dim))
                     for j in range(dim // 2)], np.float32)
    return (np.asarray(positions, np.float32)[..., None] * freq).astype(np.float64)


def rotate(x, positions, theta):
    """x [rows, heads, dim] rotated at positions [rows], in float64."""
    a = angles(positions, x.shape[-1], theta)[:, None, :]
    e, o = x[..., 0::2], x[..., 1::2]
    out = np.empty(x.shape, np.float64)
    out[..., 0::2] = e * np.cos(a) - o * np.sin(a)
    out[..., 1::2] = e * np.sin(a) + o * np.cos(a)
    return out


def attend(q, k, v, sees, scale):
    """One sequence: q [T, Hq, D] (rotated), k, v [N, Hkv, D], sees [T, N] bool, all float64. Returns O,
    LSE [Hq, T], and for error bounds sum p |v| like O and max over keys of scale * sum |q k| [Hq, T]."""
    T, hq, D = q.shape
    group = hq // k.shape[1]
    o, av = np.zeros(q.shape), np.zeros(q.shape)
    lse, size = np.full((hq, T), -np.inf), np.zeros((hq, T))
    for h in range(hq):
        kk, vv = k[:, h // group], v[:, h // group]
        for t in range(T):
            idx = np.flatnonzero(sees[t])
            if not idx.size:
                continue
            s = scale * (kk[idx] @ q[t, h])
            m = s.max()
            if m == -np.inf:
                continue
            p = np.exp(s - m)
            l = p.sum()
            o[t, h] = p @ vv[idx] / l
            av[t, h] = p @ np.abs(vv[idx]) / l
            lse[h, t] = m + np.log(l)
            size[h, t] = scale * (np.abs(kk[idx]) @ np.abs(q[t, h])).max()
    return o, lse, av, size


def accept(k, v, table, ctx, paths, accepted, lens, page, pages, max_tokens):
    """Pools [rows, width] and lengths after the accepted rows have moved; arrays are copied."""
    k, v, out = k.copy(), v.copy(), np.array(ctx)
    for s in range(len(ctx)):
        n, c = int(accepted[s]), int(ctx[s])
        if c < 0 or not 0 <= lens[s] <= max_tokens or not 0 <= n <= min(lens[s], paths.shape[1]):
            continue
        if c + lens[s] > table.shape[1] * page:
            continue
        path = [int(p) for p in paths[s, :n]]
        if any(b <= a for a, b in zip([-1] + path, path)) or any(p >= lens[s] for p in path):
            continue

        def row(logical):
            p = int(table[s, logical // page])
            return p * page + logical % page if 0 <= p < pages else -1

        moves = [(row(c + p), row(c + i)) for i, p in enumerate(path)]
        if any(f < 0 or t < 0 for f, t in moves):
            continue
        for f, t in moves:
            k[t], v[t] = k[f], v[f]
        out[s] = c + n
    return k, v, out

"""64-bit numpy restatements of the paged serving operators, a request, a token and a head at a time."""
import math

import numpy as np


def extend(table, lens, owned, free, n_free, new, drop, n_tokens, block, n_blocks, shared=0):
    """What paged_extend leaves: a dict of the arrays it writes."""
    S, M = table.shape
    table, free = table.copy(), free.copy()
    lens = [max(int(x), 0) for x in lens]
    if drop is not None:
        lens = [x - min(max(int(d), 0), x) for x, d in zip(lens, drop)]
    owned = [min(max(int(x), 0), M) for x in owned]
    top = min(max(int(n_free), 0), len(free))
    for s in range(S):
        if new[s] < 0:
            for c in range(shared, owned[s]):
                if top < len(free):
                    free[top] = table[s, c]
                    top += 1
    positions, slots = np.full(n_tokens, -1, np.int32), np.full(n_tokens, -1, np.int64)
    starts, granted, asked, have = [0], [], 0, top
    out_lens, out_owned = [], []
    stack = free.copy()
    for s in range(S):
        n = max(int(new[s]), 0)
        fits = lens[s] + n <= M * block
        need = max(0, -(-(lens[s] + n) // block) - owned[s]) if n and fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= have)
        if ok:
            for c in range(owned[s], owned[s] + need):
                top -= 1
                table[s, c] = stack[top]
            for i in range(n):
                t, p = starts[-1] + i, lens[s] + i
                if t < n_tokens:
                    positions[t] = p
                    b = int(table[s, p // block])
                    slots[t] = b * block + p % block if 0 <= b < n_blocks else -1
        granted.append(int(ok))
        starts.append(starts[-1] + n)
        out_lens.append(0 if new[s] < 0 else lens[s] + (n if ok else 0))
        out_owned.append(0 if new[s] < 0 else owned[s] + (need if ok else 0))
    return dict(table=table, free=free, n_free=np.array([top], np.int32), lens=np.array(out_lens, np.int32),
                owned=np.array(out_owned, np.int32), starts=np.array(starts, np.int32),
                granted=np.array(granted, np.int32), positions=positions, slots=slots)


def frequencies(rot, theta, scaling="none", factor=1.0, original=0, low=0.0, high=0.0):
    """Angle a position of each pair, and the magnitude."""
    if scaling == "ntk":
        theta = theta * factor ** (rot / (rot - 2))
    f = np.array([theta ** (-2.0 * i / rot) for i in range(rot // 2)])
    m = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        low, high = low or 1.0, high or 32.0
        # the pair that turns r times over the original length solves original f_i = 2 pi r
        pair = lambda r: rot / 2 * math.log(original / (2 * math.pi * r)) / math.log(theta)  # noqa: E731
        a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), rot - 1)
        for i in range(rot // 2):
            r = min(max((i - a) / max(b - a, 0.001), 0.0), 1.0)
            f[i] = f[i] * ((1 - r) + r / factor)
        m = 0.1 * math.log(factor) + 1.0
    if scaling == "wavelength":
        low, high = low or 1.0, high or 4.0
        for i in range(rot // 2):
            r = min(max((original * f[i] / (2 * math.pi) - low) / (high - low), 0.0), 1.0)
            f[i] = f[i] * (r + (1 - r) / factor)
    return f, m


def rotated(x, positions, freq, magnitude, layout, norm=None, eps=0.0):
    """x [tokens][heads][dim] in 64 bits, after the norm and the rotation."""
    x = np.asarray(x, np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    y = x.copy()
    n = len(freq)
    for i in range(n):
        a, b = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
        angle = np.asarray(positions, np.float64)[:, None] * freq[i]
        c, s = np.cos(angle) * magnitude, np.sin(angle) * magnitude
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def attend(q, k, v, table, lens, starts, scale, block, n_blocks, shared=(), max_len=None):
    """q [T][H][D], pools [n_blocks][block][KV][D].  Returns the outputs, the same sums of |v| in v's place, the largest
    scale * sum |q k| of each row's scores, and the positions it sees; rows of no sequence are NaN."""
    T, H, D = q.shape
    G = H // k.shape[2]
    out, size = np.full((T, H, D), np.nan), np.zeros((T, H, D))
    most, seen = np.zeros((T, H)), np.zeros(T, np.int64)
    S, M = table.shape
    max_len = M * block if max_len is None else max_len
    for s in range(S):
        lo, hi = (s, s + 1) if starts is None else (int(starts[s]), int(starts[s + 1]))
        for t in range(max(lo, 0), min(hi, T)):
            p = np.arange(max(min(int(lens[s]) - hi + t + 1, max_len), 0))
            ids = np.concatenate([np.asarray(shared, np.int64), table[s, len(shared):].astype(np.int64)])[p // block]
            there = (ids >= 0) & (ids < n_blocks)
            p, ids = p[there], ids[there]
            seen[t] = len(p)
            if not len(p):
                out[t] = 0.0
                continue
            for j in range(H // G):
                kk, vv = k[ids, p % block, j].astype(np.float64), v[ids, p % block, j].astype(np.float64)
                qq = q[t, j * G:(j + 1) * G].astype(np.float64)
                a = qq @ kk.T * scale
                e = np.exp(a - a.max(1, keepdims=True))
                e /= e.sum(1, keepdims=True)
                out[t, j * G:(j + 1) * G] = e @ vv
                size[t, j * G:(j + 1) * G] = e @ np.abs(vv)
                most[t, j * G:(j + 1) * G] = (np.abs(qq) @ np.abs(kk).T).max(1) * abs(scale)
    return out, size, most, seen


def verify(target, draft, tokens, starts, u, u_last):
    """(out, accepted, dropped); rows of no sequence are left -2."""
    V = target.shape[1]
    n = len(starts) - 1
    out = np.full(len(tokens), -2, np.int32)
    accepted, dropped = np.zeros(n, np.int32), np.zeros(n, np.int32)
    at = 0
    good = lambda w: np.where(np.isfinite(w) & (w > 0), w, 0.0)  # noqa: E731
    for s in range(n):
        lo, hi = int(starts[s]), int(starts[s + 1])
        if hi <= lo:
            continue
        drafted, a = hi - lo - 1, 0
        while a < drafted:
            x = int(tokens[lo + a + 1])
            if not 0 <= x < V:
                break
            q = 1.0 if draft is None else float(draft[at + a, x])
            if not float(u[at + a]) * q < float(target[lo + a, x]):
                break
            a += 1
        p = target[lo + a].astype(np.float64)
        w = good(p)
        if a < drafted:
            if draft is not None:
                left = good(p - draft[at + a].astype(np.float64))
            else:
                left = w.copy()
                if 0 <= int(tokens[lo + a + 1]) < V:
                    left[int(tokens[lo + a + 1])] = 0.0
            if left.sum() > 0:
                w = left
        out[lo:hi] = -1
        out[lo:lo + a] = tokens[lo + 1:lo + 1 + a]
        run = np.cumsum(w)
        if run[-1] > 0:
            passed = np.nonzero((run > float(u_last[s]) * run[-1]) & (w > 0))[0]
            out[lo + a] = passed[0] if len(passed) else np.nonzero(w)[0][-1]
        accepted[s], dropped[s] = a, drafted - a
        at += drafted
    return out, accepted, dropped

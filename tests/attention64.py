"""Rotary positions and attention in 64 bits, with bounds on what f32 sums and bf16 operands may add.

U = 2^-24 is f32's rounding, B = 2^-8 bf16's (both relative, half a step).  Scores are f32 sums of dim exact products: each
is off by at most (dim + 2) U times the sum of the products' magnitudes, and the exponent that is formed from it by
another 4 U of its own size and of lse's.  `slack` is that bound on the exponents: a weight is off by e^slack - 1 of itself."""
import numpy as np

U, B = 2.0 ** -24, 2.0 ** -8


def sequences(starts, n):
    """(first row, rows) of each, starts outside [0, n] counting as the nearer of the two."""
    s = np.clip(np.asarray(starts, np.int64), 0, n)
    return [(int(a), max(0, int(b - a))) for a, b in zip(s[:-1], s[1:])]


def weights(q, k, scale, seen):
    """Of q [m][dim] and k [n][dim]: p, lse and slack; seen [m][n]."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(seen, scale * (np.where(np.isfinite(q), q, 0) @ np.where(np.isfinite(k), k, 0).T), -np.inf)
    mag = scale * (np.abs(q) @ np.abs(k).T)
    top = s.max(1, initial=-np.inf)
    top = np.where(np.isfinite(top), top, 0.0)
    e = np.exp(s - top[:, None])
    total = e.sum(1)
    with np.errstate(divide="ignore"):
        lse = np.where(total > 0, top + np.log(total), -np.inf)
    p = e / np.where(total > 0, total, 1.0)[:, None]
    mag = np.where(seen, mag, 0.0).max(1, initial=0.0)
    slack = (q.shape[1] + 2) * U * mag + 4 * U * (np.where(np.isfinite(lse), np.abs(lse), 0) + mag + 1)
    return p, lse, slack


def attend(q, k, v, scale, seen):
    """out, lse of one head and the bounds of both (out's without its last rounding)."""
    p, lse, slack = weights(q, k, scale, seen)
    n = max(1, k.shape[0])
    mag = p @ np.abs(v)
    # p's rounding for the product, the exponents' error in p and in their sum, the sums over keys
    return p @ v, lse, (B + 2.2 * slack[:, None] + 2 * (n + 8) * U) * mag, 1.1 * slack + (n + 8) * U + 2 * U * np.where(np.isfinite(lse), np.abs(lse), 0)


def packed(q, k, v, starts, scale, causal):
    """q [n][heads][dim], k, v [n][kv][dim] -> out [n][heads][dim], lse [heads][n], and their bounds."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out, lse = np.zeros((n, heads, dim)), np.full((heads, n), -np.inf)
    eo, el = np.zeros_like(out), np.zeros_like(lse)
    for at, m in sequences(starts, n):
        r = slice(at, at + m)
        seen = np.tril(np.ones((m, m), bool)) if causal else np.ones((m, m), bool)
        for h in range(heads if m else 0):
            out[r, h], lse[h, r], eo[r, h], el[h, r] = attend(q[r, h], k[r, h // group], v[r, h // group], scale, seen)
    return out, lse, eo, el


def packed_grad(q, k, v, out, lse, dout, starts, scale, causal):
    """dq, dk, dv and their bounds, from the forward pass's out and lse as they are (dout as the products take it)."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    grads = [np.zeros_like(x) for x in (q, k, v)]
    bounds = [np.zeros_like(x) for x in (q, k, v)]
    for at, m in sequences(starts, n):
        r = slice(at, at + m)
        seen = np.tril(np.ones((m, m), bool)) if causal else np.ones((m, m), bool)
        for h in range(heads if m else 0):
            a, b, c, d = q[r, h], k[r, h // group], v[r, h // group], dout[r, h]
            s = scale * (a @ b.T)
            p = np.where(seen, np.exp(np.where(seen, s, -np.inf) - lse[h, r][:, None]), 0.0)
            mag = np.where(seen, scale * (np.abs(a) @ np.abs(b).T), 0.0).max(1)
            slack = ((dim + 2) * U * mag + 4 * U * (np.abs(lse[h, r]) + mag + 1))[:, None] * 1.1
            delta = (d * out[r, h]).sum(1, keepdims=True)
            dp = d @ c.T
            ds = p * (dp - delta)
            # of dp - delta: f32 sums of dim products each
            dd = (dim + 2) * U * (np.abs(d) @ np.abs(c).T + (np.abs(d) * np.abs(out[r, h])).sum(1, keepdims=True)) + 2 * U * np.abs(dp - delta)
            eds = np.abs(ds) * (B + slack) + 1.01 * p * dd
            sums = (m * group + 8) * U
            grads[0][r, h] += scale * ds @ b
            bounds[0][r, h] += scale * (eds + sums * np.abs(ds)) @ np.abs(b)
            grads[1][r, h // group] += scale * ds.T @ a
            bounds[1][r, h // group] += scale * (eds + sums * np.abs(ds)).T @ np.abs(a)
            grads[2][r, h // group] += p.T @ d
            bounds[2][r, h // group] += (p * (B + slack + sums)).T @ np.abs(d)
    return grads, bounds


def cache_positions(starts, lengths, n):
    """(sequence, first row, rows, position of the first row) of each sequence's new rows."""
    return [(s, at, m, int(lengths[s]) - m) for s, (at, m) in enumerate(sequences(starts, n))]


def paged(q, k_cache, v_cache, starts, lengths, table, scale):
    """q [n][heads][dim] over caches [pages][kv][page][dim] -> as packed()."""
    n, heads, dim = q.shape
    pages, kv, page, _ = k_cache.shape
    group = heads // kv
    out, lse = np.zeros((n, heads, dim)), np.full((heads, n), -np.inf)
    eo, el = np.zeros_like(out), np.zeros_like(lse)
    for s, at, m, pos in cache_positions(starts, lengths, n):
        length = min(max(0, int(lengths[s])), table.shape[1] * page)
        used = table[s, :-(-length // page)] if length else table[s, :0]
        there = np.repeat((used >= 0) & (used < pages), page)[:length]
        where = np.where((used >= 0) & (used < pages), used, 0)
        for h in range(heads if m and length else 0):
            k, v = (c[where, h // group].reshape(-1, dim)[:length] for c in (k_cache, v_cache))
            k, v = (np.where(there[:, None], x, 0.0) for x in (k, v))
            seen = (np.arange(length)[None] <= pos + np.arange(m)[:, None]) & there[None]
            r = slice(at, at + m)
            out[r, h], lse[h, r], eo[r, h], el[h, r] = attend(q[r, h], k, v, scale, seen)
    return out, lse, eo, el


def frequencies(rot, base=10000.0):
    return base ** (-2.0 * np.arange(rot // 2) / max(rot, 1))


def rope(x, positions, f, heads, dim, first, interleaved, inverse, magnitude):
    """x [rows][width] turned; f: radians per position of each pair."""
    y = np.array(x, np.float64)
    pairs = len(f)
    t = positions.astype(np.float64)[:, None] * f * (-1.0 if inverse else 1.0)
    c, s = magnitude * np.cos(t), magnitude * np.sin(t)
    for h in range(heads):
        at = first + h * dim
        i = at + (2 * np.arange(pairs) if interleaved else np.arange(pairs))
        j = i + (1 if interleaved else pairs)
        a, b = x[:, i].astype(np.float64), x[:, j].astype(np.float64)
        y[:, i], y[:, j] = a * c - b * s, a * s + b * c
    return y

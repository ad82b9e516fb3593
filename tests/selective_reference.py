"""Plain forms, in 64 bits, of the append with rotation and key bounds, the selection of blocks and attention over them."""

import numpy as np

FIRST_ONLY = -1  # (an entry that has ended)


def rotate(x, positions, inv_freq, interleaved):
    """x [tokens, heads, d] float64 turned by its position."""
    out = x.copy()
    n = len(inv_freq)
    if n == 0:
        return out
    angle = positions.astype(np.float64)[:, None, None] * inv_freq.astype(np.float64)
    c, s = np.cos(angle), np.sin(angle)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    a, b = x[..., first], x[..., second]
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    return out


def partners(x, n, interleaved):
    """|a| + |b| of the pair that each rotated element belongs to, 0 for the others."""
    out = np.zeros_like(x)
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    both = np.abs(x[..., first]) + np.abs(x[..., second])
    out[..., first] = out[..., second] = both
    return out


def scores(q, bounds):
    """q [group, d], bounds [n, 2, d] float64 -> [n]; what is not a number ranks as infinity."""
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.einsum("gd,nd->gn", np.maximum(q, 0), bounds[:, 1]) + np.einsum("gd,nd->gn", np.minimum(q, 0), bounds[:, 0])
        s = np.where(np.isnan(s), np.inf, s).max(0)
    return s


def choose(score, n, budget, first, last):
    """Columns of the n blocks, ascending, -1 behind them."""
    out = np.full(budget, -1, np.int64)
    if n <= budget:
        out[:n] = np.arange(n)
        return out
    ends = [c for c in range(n) if c < first or c >= n - last]
    rest = [c for c in range(n) if first <= c < n - last]
    rest.sort(key=lambda c: (-score[c], c))
    out[:] = sorted(ends + rest[: budget - len(ends)])
    return out


def select(q, bounds, tables, lens, positions, bs, budget, first, last):
    """q [rows, width, hq, d], bounds [pool, hkv, 2, d], positions [rows, width] or None -> [rows, width, hkv, budget]."""
    rows, width, hq, _ = q.shape
    hkv = bounds.shape[1]
    group = hq // hkv
    out = np.full((rows, width, hkv, budget), -1, np.int64)
    for b in range(rows):
        for t in range(width):
            seen = visible(lens, positions, b, t)
            n = max(0, -(-seen // bs))
            for h in range(hkv):
                held = bounds[tables[b, :n], h]
                score = scores(q[b, t, h * group:(h + 1) * group], held) if n > budget else None
                out[b, t, h] = choose(score, n, budget, first, last)
    return out


def visible(lens, positions, b, t):
    return int(lens[b]) if positions is None else max(0, min(int(lens[b]), int(positions[b, t]) + 1))


def attend(q, k, v, tables, lens, positions, selected, scale, bs, gamma, weight_bits):
    """Softmax over the listed blocks, and the error that rounding may make of it: scores are sums of d products, off by gamma * sum |q k| at
    most; a weight follows its score (twice: numerator and sum) and is kept to 2^-weight_bits; sums of n terms are off by n * 2^-23 of their terms' sizes."""
    rows, width, hq, d = q.shape
    hkv = k.shape[2]
    group = hq // hkv
    out, tol = np.zeros((rows, width, hq, d)), np.zeros((rows, width, hq, d))
    for b in range(rows):
        for t in range(width):
            seen = visible(lens, positions, b, t)
            for h in range(hkv):
                place = [(c, p) for c in selected[b, t, h] if c >= 0 and c < tables.shape[1] for p in range(c * bs, min((c + 1) * bs, seen))]
                if not place:
                    continue
                block = tables[b, [c for c, _ in place]]
                at = np.array([p - c * bs for c, p in place])
                kk, vv = k[block, at, h], v[block, at, h]
                for g in range(h * group, (h + 1) * group):
                    s = scale * (kk @ q[b, t, g])
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[b, t, g] = w @ vv
                    slip = abs(scale) * gamma * (np.abs(kk) @ np.abs(q[b, t, g])).max()
                    tol[b, t, g] = (w @ np.abs(vv)) * (2 * slip * (1 + slip) + 2.0 ** -weight_bits + len(place) * 2.0 ** -23 + 2.0 ** -20)
    return out, tol

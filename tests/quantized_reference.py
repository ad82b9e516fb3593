"""The 8-bit paged cache in plain NumPy, in 64 bits: append, attention, and how far a kernel's sums may be from the latter."""

from __future__ import annotations

import math

import numpy as np
import torch

LOW, HIGH, LARGEST = -117, 119, 448.0
_VALUES = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).to(torch.float64).numpy()  # what a byte stands for
_MAGNITUDES = _VALUES[:127]  # 0 .. 448, growing


def values(codes):
    return _VALUES[codes]


def nearest(x):
    """Bytes of the e4m3 numbers next to x (ties to the even one), magnitudes over 448 held there, NaN kept."""
    size = np.abs(x)
    size = np.where(np.isnan(size), 0.0, np.minimum(size, LARGEST))
    above = np.minimum(np.searchsorted(_MAGNITUDES, size, side="left"), 126)
    below = np.maximum(above - 1, 0)
    up, down = _MAGNITUDES[above] - size, size - _MAGNITUDES[below]
    code = np.where(up < down, above, np.where(down < up, below, np.where(above % 2 == 0, above, below)))
    code = np.where(_MAGNITUDES[above] == size, above, code).astype(np.uint8)
    code = code | (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isnan(x), np.uint8(127), code)


def scale_for(largest):
    e = LOW
    if largest > 0:
        e = math.frexp(largest)[1] - 10
        while largest > LARGEST * 2.0 ** e:
            e += 1
    return 2.0 ** min(max(e, LOW), HIGH)


def append(codes, scale, new, tokens, block_size):
    """In place: codes [blocks, bs, hkv, d] bytes, scale [blocks, hkv]; new [n, hkv, d] float64 with tokens[i] = (block id, offset) or None."""
    runs = {}
    for i, at in enumerate(tokens):
        if at is not None:
            runs.setdefault(at[0], []).append((i, at[1]))
    for block, members in runs.items():
        for h in range(codes.shape[2]):
            x = np.stack([new[i, h] for i, _ in members])
            finite = np.abs(x[np.isfinite(x)])
            wanted = scale_for(finite.max() if finite.size else 0.0)
            begins = any(o == 0 for _, o in members)
            now = wanted if begins else max(wanted, scale[block, h])
            if not begins and now > scale[block, h]:
                codes[block, :, h] = nearest(values(codes[block, :, h]) * (scale[block, h] / now))
            for (i, o), row in zip(members, x):
                codes[block, o, h] = nearest(row / now)
            scale[block, h] = now


def gather(codes, scale, table, n):
    """float64 [n, hkv, d]: the values of a row's first n tokens."""
    blocks = np.asarray(table)[: -(-n // codes.shape[1])]
    x = values(codes[blocks]) * scale[blocks][:, None, :, None].astype(np.float64)
    return x.reshape(-1, *codes.shape[2:])[:n]


def attend(q, k, v, seen, scale):
    """softmax(scale q k^T) v in float64 for one row: q [t, hq, d], k, v [n, hkv, d], seen [t, n]; no key seen gives zeros."""
    t, hq, d = q.shape
    groups = hq // k.shape[1]
    out = np.zeros((t, hq, d))
    for j in range(hq):
        s = np.where(seen, (q[:, j] @ k[:, j // groups].T) * scale, -np.inf)
        top = s.max(1, keepdims=True) if s.shape[1] else np.full((t, 1), -np.inf)
        w = np.exp(s - np.where(np.isfinite(top), top, 0.0))
        w[~np.broadcast_to(seen, w.shape)] = 0.0
        total = w.sum(1, keepdims=True)
        out[:, j] = (w @ np.where(seen.any(0)[:, None], v[:, j // groups], 0.0)) / np.where(total > 0, total, 1.0)
    return out


def tolerance(q, k, v, scale, term_bits=22):
    """Bound on |kernel - attend| for one row, from what the kernels round:

    * a score is a sum of d products that are exact in f32, taken 16 at a time: every step may cut a last place (2^-23) of a partial sum of
      at most S = scale * max sum |q k|, and the two factors behind the sum round twice: an absolute error of (d / 16 + 2) 2^-23 S;
    * a weight's relative error is that times 1 (d exp(s) = exp(s) ds), 2^-22 each of the exponent's two roundings (times |s| <= S) and of
      ex2.approx, and 2^-term_bits of its terms (two of f16: 22, two of bf16: 16, five of e4m3: 20); in numerator and denominator;
    * (f32 queries as five e4m3 terms, 2^-20: inside the same, S / 2^20 < (d / 16 + 2) S / 2^23 for d >= 128)
    * the weighted sum takes two products (high and low term) per 16 keys, 2^-23 of a partial sum cut each time, the sum of
      the weights one addition per key: (n / 8 + n) 2^-23; merging warps and CTAs adds a few.
    All of it relative to the largest |v|, which bounds the weighted mean."""
    n, d = k.shape[0], q.shape[2]
    if n == 0:
        return 0.0
    groups = q.shape[1] // k.shape[1]
    most = max(float((np.abs(q[:, j]) @ np.abs(k[:, j // groups]).T).max()) for j in range(q.shape[1])) * abs(scale) if q.size else 0.0
    weight = (d / 16 + 2) * 2.0 ** -23 * most + 2.0 ** -22 * (2 + 2 * most) + 2.0 ** -term_bits
    return float(np.abs(v).max()) * (2 * weight + (n / 8 + n + 64) * 2.0 ** -23)

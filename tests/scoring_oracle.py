"""Attention with a cap, a bias or ranges over a paged cache, in 64 bits and one row after the other."""
import numpy as np

import paged_oracle as po


def mask_of(i, length, window, sinks, ranges=None):
    j = np.arange(length)
    low, upto = (0, i + 1) if ranges is None else (max(int(ranges[0]), 0), min(int(ranges[1]), length))
    if i < 0:
        return np.zeros(length, bool)
    if window:
        low = max(low, i + 1 - window)
    if window == 0 and ranges is None:
        sinks = 0
    return (j < upto) & ((j >= low) | (j < sinks))


def attention(pool, q, starts, scale, *, cap=0.0, slopes=None, ranges=None, window=0, sinks=0, gate=None):
    """(output, lse, their bounds by the roundings of the kernels); rows that no sequence has are NaN."""
    total, hq, d = q.shape
    g = hq // pool.heads
    out, lse, bound, lse_bound = np.full((total, hq, d), np.nan), np.full((total, hq), np.nan), np.full((total, hq, d), np.nan), np.full((total, hq), np.nan)
    u_k = po.HALF_STEP if pool.mode in (1, 3) else 0.0
    u_v = po.HALF_STEP if pool.mode in (2, 3) else 0.0
    u_q = po.HALF_STEP if q.dtype == np.float32 else 0.0
    q = q.astype(np.float64)
    for s, length in enumerate(pool.lengths):
        n = int(starts[s + 1] - starts[s])
        for h in range(pool.heads):
            k, v = pool.rows(s, h, 0), pool.rows(s, h, 1)
            for t in range(n):
                row, i = int(starts[s]) + t, length - n + t
                m = mask_of(i, length, window, sinks, None if ranges is None else ranges[row])
                for e in range(h * g, (h + 1) * g):
                    if not m.any():
                        out[row, e], lse[row, e], bound[row, e], lse_bound[row, e] = 0.0, -np.inf, 0.0, 0.0
                        continue
                    x = k[m] @ q[row, e] * scale
                    if cap:
                        x = cap * np.tanh(x / cap)
                    far = 0.0
                    if slopes is not None:
                        away_from = np.abs(i - np.flatnonzero(m))
                        x = x - float(slopes[e]) * away_from
                        far = abs(float(slopes[e])) * away_from.max()
                    top = x.max()
                    p = np.exp(x - top)
                    total_p = p.sum()
                    p /= total_p
                    o = p @ v[m]
                    lse[row, e] = top + np.log(total_p)
                    # as without a cap (paged_oracle.attention): no slope of cap * tanh(x / cap) is above 1.  A tanh is off by 3e-7 (2^-21.6), its product with the cap by a rounding:
                    # 2^-20 of the cap together; the bias and the sum with it by three roundings of the largest: 2^-22 of it
                    away = (np.abs(k[m]) @ np.abs(q[row, e])).max() * scale * (u_k + u_q + 2.0 ** -20) + cap * 2.0 ** -20 + far * 2.0 ** -22
                    b = (p @ np.abs(v[m])) * (np.expm1(2 * away) + 2 * po.HALF_STEP + u_v + 2.0 ** -18)
                    if u_v:
                        b = b + 2.0 ** -17 * (1 + 2.0 ** -10) * p.max() * pool.whole_values(s, h, length)[m].sum(0)
                    if gate is not None:
                        f = 1 / (1 + np.exp(-gate[row, e].astype(np.float64)))
                        o, b = o * f, b * f + np.abs(o) * 2.0 ** -20
                    out[row, e] = o
                    bound[row, e] = b + po.HALF_STEP * np.abs(o) + 2.0 ** -24
                    # exponentials and their sum: 2^-18 (a row's 64 columns of a tile and its tiles); maximum and logarithm: 2^-21 of the value, which the largest score bounds too
                    lse_bound[row, e] = away + 2.0 ** -18 + 2.0 ** -20 * (abs(lse[row, e]) + abs(top))
    return out, lse, bound, lse_bound

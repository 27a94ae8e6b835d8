"""Plain implementations, in 64 bits and one row after the other, of the operators over a paged cache, and the pools and batches their tests use."""
import numpy as np
import torch

from miinfer_b200 import kv, paged

HALF_STEP = 2.0 ** -11      # fp16 rounding, relative to the value


class Pool:
    """A pool with random rows on the host and on the device; sequences' pages scattered over it."""

    def __init__(self, rng, lengths, *, d, heads, page, mode, qblock, spare=2, k_std=1.0, extra_columns=1, capacity=None):
        self.d, self.heads, self.page, self.mode, self.qblock = d, heads, page, mode, qblock
        self.lengths = list(lengths)
        room = self.lengths if capacity is None else [capacity] * len(self.lengths)
        need = [-(-n // page) for n in room]
        self.pages = sum(need) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(need), max(need, default=0) + extra_columns), -7, np.int32)     # entries past a length are never read
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.spare = order[at:]
        shape = (self.pages, heads, page, d)
        self.k, self.ks = self._side(rng, shape, mode in (1, 3), k_std)
        self.v, self.vs = self._side(rng, shape, mode in (2, 3), 1.0)

    def _side(self, rng, shape, q8, std):
        x = rng.standard_normal(shape, dtype=np.float32) * std
        if not q8:
            return x.astype(np.float16), None
        b = x.reshape(*shape[:3], -1, self.qblock)
        scale = (np.abs(b).max(-1) / 127).astype(np.float16)
        return np.clip(np.rint(b / scale.astype(np.float32)[..., None]), -128, 127).astype(np.int8).reshape(shape), scale

    def rows(self, s, h, side, length=None):
        """K (0) or V (1) of one sequence's kv head, float64 [length][d]."""
        plane, scales = (self.k, self.ks) if side == 0 else (self.v, self.vs)
        n = self.lengths[s] if length is None else length
        pages = self.table[s, :-(-n // self.page)]
        x = plane[pages, h].reshape(-1, self.d)[:n].astype(np.float64)
        if scales is None:
            return x
        sc = scales[pages, h].reshape(-1, self.d // self.qblock)[:n].astype(np.float64)
        return (x.reshape(n, self.d // self.qblock, self.qblock) * sc[:, :, None]).reshape(n, self.d)

    def whole_values(self, s, h, length):
        """|int8 values| of a sequence's kv head times the largest scale of their block of dims, float64 [length][d]."""
        pages = self.table[s, :-(-length // self.page)]
        q = np.abs(self.v[pages, h].reshape(-1, self.d)[:length].astype(np.float64))
        most = self.vs[pages, h].reshape(-1, self.d // self.qblock)[:length].astype(np.float64).max(0)
        return q * np.repeat(most, self.qblock)

    def place(self, s, j):
        return self.table[s, j // self.page], j % self.page

    def upload(self):
        dev = lambda a: None if a is None else torch.from_numpy(a).cuda()
        self.dev = [dev(a) for a in (self.k, self.ks, self.v, self.vs)]
        self.table_dev = torch.from_numpy(self.table).cuda()
        return paged.PagedView.of(*self.dev, kv.KvCacheQuantMode(self.mode))


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def batch_of(pool, tokens, *, pad_rows=0, starts=None, **bounds):
    """The batch of `tokens[s]` newest tokens of every sequence; pad_rows: rows of the activations behind the last sequence's."""
    starts = np.concatenate([[0], np.cumsum(tokens)]) if starts is None else np.asarray(starts)
    args = dict(total_tokens=int(starts[-1]) + pad_rows, max_tokens=max(int(max(tokens)), 1), max_length=max(max(pool.lengths), 1), total_length=sum(pool.lengths))
    args.update(bounds)
    return paged.PagedBatch(pool.table_dev, ints(starts), ints(pool.lengths), **args), starts


def sees(i, j, window, sinks):
    return j <= i and (window == 0 or j > i - window or j < sinks)


def mask_of(i, length, window, sinks):
    j = np.arange(length)
    m = j <= i
    if window:
        m &= (j > i - window) | (j < sinks)
    return m


def attention(pool, q, starts, scale, window=0, sinks=0, gate=None):
    """(output, lse, error bound of the output by the roundings of the kernels), rows that no sequence has left at NaN."""
    total, hq, d = q.shape
    g = hq // pool.heads
    out, lse, bound = np.full((total, hq, d), np.nan), np.full((total, hq), np.nan), np.full((total, hq, d), np.nan)
    u_k = HALF_STEP if pool.mode in (1, 3) else 0.0
    u_v = HALF_STEP if pool.mode in (2, 3) else 0.0
    u_q = HALF_STEP if q.dtype == np.float32 else 0.0
    q = q.astype(np.float64)
    for s, length in enumerate(pool.lengths):
        n = int(starts[s + 1] - starts[s])
        for h in range(pool.heads):
            k, v = pool.rows(s, h, 0), pool.rows(s, h, 1)
            for t in range(n):
                m = mask_of(length - n + t, length, window, sinks)
                row = starts[s] + t
                for e in range(h * g, (h + 1) * g):
                    if not m.any():
                        out[row, e], lse[row, e], bound[row, e] = 0.0, -np.inf, 0.0
                        continue
                    x = k[m] @ q[row, e] * scale
                    top = x.max()
                    p = np.exp(x - top)
                    total_p = p.sum()
                    p /= total_p
                    o = p @ v[m]
                    lse[row, e] = top + np.log(total_p)
                    # scores: K and q rounded, fp32 sums of the products (2^-20 of their magnitudes: d terms, each link at most a unit of 2^-24 and half of
                    # them below that on average); the weights' sum and the weights move with them; weights and V are rounded once, the sum of
                    # rounded weights divides
                    away = (np.abs(k[m]) @ np.abs(q[row, e])).max() * scale * (u_k + u_q + 2.0 ** -20)
                    b = (p @ np.abs(v[m])) * (np.expm1(2 * away) + 2 * HALF_STEP + u_v + 2.0 ** -18)
                    # int8 values: a weight times its value scale may be a whole number of 65535ths of the largest weight times the largest scale of the block
                    # (of a tile: no more than of all), each off by half of one, and multiplies a whole number of at most 128
                    if u_v:
                        b = b + 2.0 ** -17 * (1 + 2.0 ** -10) * p.max() * pool.whole_values(s, h, length)[m].sum(0)
                    if gate is not None:
                        f = 1 / (1 + np.exp(-gate[row, e].astype(np.float64)))
                        o, b = o * f, b * f + np.abs(o) * 2.0 ** -20
                    out[row, e] = o
                    bound[row, e] = b + HALF_STEP * np.abs(o) + 2.0 ** -24
    return out, lse, bound


def weights(pool, q, lse, starts, scale, window=0, sinks=0, observe=0):
    """(what is added per sequence [kv_head][length], its bound): fp32 arithmetic on scores."""
    hq = q.shape[1]
    g = hq // pool.heads
    got, bounds = [], []
    q = q.astype(np.float64)
    for s, length in enumerate(pool.lengths):
        n = int(starts[s + 1] - starts[s])
        a, b = np.zeros((pool.heads, length)), np.zeros((pool.heads, length))
        for h in range(pool.heads):
            k = pool.rows(s, h, 0)
            for t in range(n - min(n, observe) if observe else 0, n):
                m = mask_of(length - n + t, length, window, sinks)
                for e in range(h * g, (h + 1) * g):
                    l = float(lse[starts[s] + t, e])
                    if l == -np.inf:
                        continue
                    row = q[starts[s] + t, e]
                    x = k @ row * scale
                    w = np.where(m, np.exp(np.minimum(x - l, 700)), 0.0)
                    # a score's products and sums, and the rounding of score and statistics in units of their magnitude
                    away = (np.abs(k) @ np.abs(row)) * scale * 2.0 ** -20 + (np.abs(x) + abs(l)) * 2.0 ** -22
                    a[h] += w
                    b[h] += w * (np.expm1(away) + 2.0 ** -21)
        got.append(a)
        bounds.append(b + np.abs(a) * 2.0 ** -20)
    return got, bounds


def evict(w, length, keep, sinks, recent):
    """The positions that stay, of one sequence and kv head."""
    if length <= keep:
        return np.arange(length)
    rank = np.array([(-np.inf if np.isnan(x) else float(x)) for x in w[:length]])
    nan = np.isnan(w[:length])
    rank_key = sorted(range(length), key=lambda j: (not (j < sinks or j >= length - recent), nan[j], -rank[j], j))
    return np.array(sorted(rank_key[:keep]))

"""A bias by distance of any steepness: off by a fraction of itself at every position, and by nothing at the token's own."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from test_scoring_gpu import dev, status  # noqa: F401
from miinfer_b200 import paged
import scoring_oracle as so

pytestmark = pytest.mark.gpu


def rows(pool, q, starts, scale, cap, slopes, ranges):
    """(output, lse, their bounds): as scoring_oracle.attention's, but that every position's bias counts with its own error, 2^-22 of itself (a slope in log2 units is off by two roundings,
    its product with a distance and the sum by one each), and not with the farthest one's."""
    with np.errstate(over="ignore", invalid="ignore"):      # (the bounds that are not taken)
        out, lse = so.attention(pool, q, starts, scale, cap=cap, slopes=slopes, ranges=ranges)[:2]
    bound, lse_bound = np.zeros_like(out), np.zeros_like(lse)
    u_k = po.HALF_STEP if pool.mode in (1, 3) else 0.0
    u_v = po.HALF_STEP if pool.mode in (2, 3) else 0.0
    u_q = po.HALF_STEP if q.dtype == np.float32 else 0.0
    q, g = q.astype(np.float64), q.shape[1] // pool.heads
    for s, length in enumerate(pool.lengths):
        n = int(starts[s + 1] - starts[s])
        for e in range(q.shape[1]):
            k, v = pool.rows(s, e // g, 0), pool.rows(s, e // g, 1)
            for t in range(n):
                row, i = int(starts[s]) + t, length - n + t
                m = so.mask_of(i, length, 0, 0, None if ranges is None else ranges[row])
                if not m.any():
                    continue
                x = k[m] @ q[row, e] * scale
                x = cap * np.tanh(x / cap) if cap else x
                far = float(slopes[e]) * np.abs(i - np.flatnonzero(m))
                x = x - far
                p = np.exp(x - x.max())
                p /= p.sum()
                away = (np.abs(k[m]) @ np.abs(q[row, e])) * scale * (u_k + u_q + 2.0 ** -20) + cap * 2.0 ** -20 + np.abs(far) * 2.0 ** -22
                # all scores off at once, each to its side: ln(sum p_j exp(+-away_j)); a weight far below 1 stays so, whatever its own error
                w = p * np.exp(np.minimum(away, 700.0))
                moved = np.log(np.maximum(w.sum(), 1.0))
                assert np.isfinite(moved) and moved < 1.0          # (the inputs leave something to test)
                lse_bound[row, e] = moved + 2.0 ** -18 + 2.0 ** -20 * (abs(lse[row, e]) + abs(x.max()))
                b = (w * np.exp(moved) - p) @ np.abs(v[m]) + (p @ np.abs(v[m])) * (2 * po.HALF_STEP + u_v + 2.0 ** -18)
                if u_v:
                    b = b + 2.0 ** -17 * (1 + 2.0 ** -10) * p.max() * pool.whole_values(s, e // g, length)[m].sum(0)
                bound[row, e] = b + po.HALF_STEP * np.abs(out[row, e]) + 2.0 ** -24
    return out, lse, bound, lse_bound


STEEP = np.array([0.0, 1.0, 7.3, 100.0, 1234.5, 1.0e4, 1.0e6, 1.0e9], np.float32)


@pytest.mark.parametrize("cap", [0.0, 60.0, 6.0, 0.7])
@pytest.mark.parametrize("kind", [None, "prefix", "behind"])
@pytest.mark.parametrize("d,mode", [(128, 0), (256, 0), (128, 3)])
@pytest.mark.parametrize("tokens", [[130, 41, 70], [1, 1, 1]])
def test_steep_slopes(cuda, status, cap, kind, d, mode, tokens):
    """Causal rows, rows that see both sides of themselves, rows whose own position is the last or the first that they see."""
    rng = np.random.default_rng(d + mode)
    pool = po.Pool(rng, [321, 41, 200], d=d, heads=2, page=16, mode=mode, qblock=32)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens)
    slopes = np.resize(STEEP, 8)
    ranges = None
    if kind is not None:
        of = []
        for n, length in zip(tokens, pool.lengths):
            i = np.arange(length - n, length)
            of.append(np.stack([np.zeros(n, int), np.full(n, length)], 1) if kind == "prefix" else np.stack([i, np.full(n, length)], 1))
        ranges = np.concatenate(of).astype(np.int32)
    q = (1.5 * rng.standard_normal((batch.total_tokens, 8, d))).astype(np.float16)
    out, lse = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape[:2], device="cuda")
    scoring = paged.PagedScoring(cap=cap, slopes=dev(slopes), ranges=None if ranges is None else dev(ranges))
    paged.launch_paged_attention(view, batch, dev(q), out, query_heads=8, scale=d ** -0.5, lse=lse, scoring=scoring, workspace=paged.paged_workspace(view, batch, 8, scoring=scoring))
    want, want_lse, bound, lse_bound = rows(pool, q, starts, d ** -0.5, cap, slopes, ranges)
    off = np.abs(lse.cpu().numpy() - want_lse)
    worst = np.unravel_index(np.argmax(off - lse_bound), off.shape)
    assert (off <= lse_bound).all(), (worst, float(slopes[worst[1]]), off[worst], lse_bound[worst])
    off = np.abs(out.cpu().numpy() - want)
    worst = np.unravel_index(np.argmax(off - bound), off.shape)
    assert (off <= bound).all(), (worst, float(slopes[worst[1]]), off[worst], bound[worst])
    assert int(status) == 0


@pytest.mark.parametrize("slope", [1.0e30, -1.0e30, 1.0e20])
@pytest.mark.parametrize("tokens", [[130, 41], [1, 1]])
def test_the_steepest_slopes(cuda, status, slope, tokens):
    """Nothing but the nearest position, or the farthest, has a weight: the output is its value."""
    rng = np.random.default_rng(3)
    pool = po.Pool(rng, [321, 41], d=128, heads=1, page=16, mode=0, qblock=32)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens)
    q = (1.5 * rng.standard_normal((batch.total_tokens, 2, 128))).astype(np.float16)
    out = torch.zeros(q.shape, dtype=torch.float16, device="cuda")
    scoring = paged.PagedScoring(slopes=dev(np.full(2, slope, np.float32)))
    paged.launch_paged_attention(view, batch, dev(q), out, query_heads=2, scale=0.09, scoring=scoring, workspace=paged.paged_workspace(view, batch, 2, scoring=scoring))
    got = out.cpu().numpy()
    for s, length in enumerate(pool.lengths):
        for t in range(tokens[s]):
            at = length - tokens[s] + t if slope > 0 else 0
            assert np.array_equal(got[int(starts[s]) + t], np.repeat(pool.rows(s, 0, 1)[at:at + 1], 2, 0).astype(np.float16))
    assert int(status) == 0


@pytest.mark.parametrize("tokens", [[30, 1], [1, 1]])
@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("scores", [dict(cap=10.0), dict(cap=10.0, slopes=True), dict(slopes=True)])
def test_infinite_queries_stay_in_their_rows(cuda, status, tokens, act, scores):
    rng = np.random.default_rng(6)
    pool = po.Pool(rng, [90, 40], d=128, heads=2, page=16, mode=0, qblock=128)
    view = pool.upload()
    batch, _ = po.batch_of(pool, tokens)
    q = dev((1.5 * rng.standard_normal((batch.total_tokens, 4, 128))).astype(act))
    scoring = paged.PagedScoring(cap=scores.get("cap", 0.0), slopes=dev(np.array([0.5, 0.25, 2.0, 1.0], np.float32)) if "slopes" in scores else None)
    ws = paged.paged_workspace(view, batch, 4, scoring=scoring)
    clean, out = (torch.zeros(q.shape, dtype=torch.float16, device="cuda") for _ in range(2))
    paged.launch_paged_attention(view, batch, q, clean, query_heads=4, scale=0.09, workspace=ws, scoring=scoring)
    for value in (float("inf"), -float("inf")):
        q[0, 1, 5] = value
        paged.launch_paged_attention(view, batch, q, out, query_heads=4, scale=0.09, workspace=ws, scoring=scoring)
        out[0, 1] = clean[0, 1]
        assert bool(torch.isfinite(out).all())
        # the other rows' scores may be capped another way, each off by 2^-20 of the cap, and their weights and outputs are rounded to fp16 after that
        most = float(np.abs(pool.v).max())
        assert float((out.float() - clean.float()).abs().max()) <= most * (np.expm1(4 * scores.get("cap", 0.0) * 2.0 ** -20) + 4 * po.HALF_STEP)
    assert int(status) == 0

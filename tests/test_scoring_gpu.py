"""Attention over a paged cache with a cap, a bias by distance and ranges of the tokens' own, against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

import paged_oracle as po
import scoring_oracle as so
from miinfer_b200 import kv, paged

pytestmark = pytest.mark.gpu


@pytest.fixture
def status():
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.set_status_word(word)
    yield word
    kv.set_status_word(None)


dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()


def slopes_of(hq):
    return 2.0 ** (-8.0 * np.arange(1, hq + 1) / hq).astype(np.float32)


def ranges_of(rng, kind, tokens, lengths, pad_rows=0):
    """[row][2] of every token."""
    got = []
    for n, length in zip(tokens, lengths):
        i = np.arange(length - n, length)
        if kind == "documents":
            starts = np.unique(np.concatenate([[0], rng.integers(0, max(length, 1), 5)]))
            got.append(np.stack([starts[np.searchsorted(starts, i, side="right") - 1], i + 1], 1))
        elif kind == "prefix":
            p = int(rng.integers(0, length + 1))
            got.append(np.stack([np.zeros(n, int), np.where(i < p, p, i + 1)], 1))
        else:       # anything: empty ones, ones past the length, negative ones
            a, b = rng.integers(-20, length + 20, (2, n))
            got.append(np.stack([a, np.where(rng.random(n) < 0.8, a + rng.integers(0, length + 1, n), b)], 1))
    got.append(np.full((pad_rows, 2), 7))
    return np.concatenate(got).astype(np.int32).reshape(-1, 2)


def unseen(pool, tokens, starts, window, sinks, ranges):
    """Positions of every sequence that lie outside all that its tokens see: below the lowest or behind the last, and no sink."""
    for s, length in enumerate(pool.lengths):
        seen = np.zeros(length, bool)
        for t in range(tokens[s]):
            m = so.mask_of(length - tokens[s] + t, length, window, sinks, None if ranges is None else ranges[int(starts[s]) + t])
            seen |= m
        at = np.flatnonzero(seen)
        main = at[at >= sinks] if (window or ranges is not None) else at
        filled = np.zeros(length, bool)
        if len(main):
            filled[main[0]:main[-1] + 1] = True
        if window or ranges is not None:
            filled |= seen & (np.arange(length) < sinks)
            if len(at):     # a row below the sinks may be seen as one of a range: the documented extent is from the lowest to the last
                lows = []
                for t in range(tokens[s]):
                    i = length - tokens[s] + t
                    low = 0 if ranges is None else max(int(ranges[int(starts[s]) + t][0]), 0)
                    upto = i + 1 if ranges is None else min(int(ranges[int(starts[s]) + t][1]), length)
                    low = max(low, i + 1 - window) if window else low
                    if low < upto and i >= 0:
                        lows.append(low)
                if lows:
                    filled[min(lows):at[-1] + 1] = True
                filled[:min(sinks, at[-1] + 1)] = True
        yield s, np.flatnonzero(~filled)


def run(rng, pool, tokens, *, hq, cap=0.0, slopes=None, ranges=None, window=0, sinks=0, act=np.float16, out_dtype=torch.float16, gated=False, pad_rows=1, q_std=1.5, poison=True, word=None,
        **bounds):
    view = pool.upload()
    d = pool.d
    batch, starts = po.batch_of(pool, tokens, pad_rows=pad_rows, **bounds)
    total, n = batch.total_tokens, int(starts[-1])
    if poison:      # what nobody sees may be anything: rows past a length, and those outside all that a sequence's tokens see
        for s, length in enumerate(pool.lengths):
            if length % pool.page:
                for p in pool.dev:
                    if p is not None and p.dtype == torch.float16:
                        p[int(pool.table[s, length // pool.page]), :, length % pool.page:] = float("nan")
        for s, rows in unseen(pool, tokens, starts, window, sinks, ranges):
            for j in rows:
                pg, slot = pool.place(s, int(j))
                for p in pool.dev:
                    if p is not None and p.dtype == torch.float16:
                        p[pg, :, slot] = float("nan")
    q = (q_std * rng.standard_normal((total, hq, d))).astype(act)
    gate = rng.standard_normal((total, hq, d)).astype(np.float32) if gated else None
    out = torch.full((total, hq, d), 5.0, dtype=out_dtype, device="cuda")
    lse = torch.full((total, hq), 5.0, device="cuda")
    scoring = paged.PagedScoring(cap=cap, slopes=None if slopes is None else dev(slopes), ranges=None if ranges is None else dev(ranges))
    ws = paged.paged_workspace(view, batch, hq, window=window, sinks=sinks, scoring=scoring).fill_(255)
    paged.launch_paged_attention(view, batch, dev(q), out, query_heads=hq, scale=d ** -0.5, window=window, sinks=sinks, gate=None if gate is None else dev(gate), lse=lse,
                                 workspace=ws, scoring=scoring)
    want, want_lse, bound, lse_bound = so.attention(pool, q, starts, d ** -0.5, cap=cap, slopes=slopes, ranges=ranges, window=window, sinks=sinks, gate=gate)
    got, got_lse = out.cpu().numpy().astype(np.float64), lse.cpu().numpy().astype(np.float64)
    assert (got[n:] == 5.0).all() and (got_lse[n:] == 5.0).all()
    off = np.abs(got[:n] - want[:n])
    worst = np.unravel_index(np.argmax(np.nan_to_num(off - bound[:n], nan=np.inf)), off.shape)
    assert (off <= bound[:n]).all(), (worst, got[:n][worst], want[:n][worst], bound[:n][worst], float((off > bound[:n]).mean()))
    assert np.array_equal(np.isneginf(got_lse[:n]), np.isneginf(want_lse[:n]))
    fine = np.isfinite(want_lse[:n])
    off = np.abs(got_lse[:n][fine] - want_lse[:n][fine])
    assert (off <= lse_bound[:n][fine]).all(), (off.max(), lse_bound[:n][fine][np.argmax(off)])
    assert word is None or int(word) == 0
    return out, lse


SCORES = [dict(cap=4.0), dict(slopes=True), dict(cap=30.0, slopes=True), dict()]
RAGGED = [40, 9, 1, 130, 65, 7, 200], [40, 0, 1, 2, 5, 7, 33]
SINGLE = [1, 2, 15, 16, 17, 127, 128, 129, 500, 1000], [1, 1, 1, 1, 1, 0, 1, 1, 1, 1]
MODES = [(0, 32), (3, 32), (3, None), (1, 32), (2, None), (2, 32), (1, None)]


@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("scores", range(3))
@pytest.mark.parametrize("d,heads,hq,page", [(128, 2, 8, 16), (256, 2, 12, 64), (128, 3, 3, 256), (256, 1, 8, 32)])
@pytest.mark.parametrize("lengths,tokens", [RAGGED, SINGLE])
def test_caps_and_biases(cuda, status, mode, qblock, scores, d, heads, hq, page, lengths, tokens):
    rng = np.random.default_rng(1000 * mode + d + hq + scores)
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=page, mode=mode, qblock=qblock or d)
    args = dict(SCORES[scores])
    if args.pop("slopes", False):
        args["slopes"] = slopes_of(hq)
    run(rng, pool, tokens, hq=hq, gated=hq == 12, q_std=4.0, word=status, **args)


@pytest.mark.parametrize("kind", ["documents", "prefix", "any"])
@pytest.mark.parametrize("d,mode,qblock,heads,hq", [(128, 0, 128, 2, 8), (256, 3, 32, 1, 6), (128, 3, 128, 3, 3), (256, 0, 256, 2, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 5), (50, 0), (64, 70), (7, 3), (0, 100)])
@pytest.mark.parametrize("lengths,tokens", [([300, 70, 40, 130, 260, 1], [90, 1, 40, 3, 1, 1]), ([300, 70, 40, 130, 260, 1], [1, 1, 1, 0, 1, 1])])
def test_ranges(cuda, status, kind, d, mode, qblock, heads, hq, window, sinks, lengths, tokens):
    rng = np.random.default_rng(d + window + 3 * sinks + len(kind))
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=32, mode=mode, qblock=qblock)
    ranges = ranges_of(rng, kind, tokens, lengths, 1)
    scores = SCORES[(window + sinks) % 4]
    run(rng, pool, tokens, hq=hq, ranges=ranges, window=window, sinks=sinks, cap=scores.get("cap", 0.0), slopes=slopes_of(hq) if "slopes" in scores else None, word=status)


@pytest.mark.parametrize("tokens", [[3, 2, 4, 1], [30, 2, 4, 1], [1, 1, 1, 1]])
@pytest.mark.parametrize("d,mode", [(128, 0), (256, 3)])
def test_rows_that_see_nothing(cuda, status, tokens, d, mode):
    """Every range of a sequence empty, past its length or before its first position; the others' as they are."""
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [200, 70, 5, 64], d=d, heads=2, page=16, mode=mode, qblock=32)
    ranges = ranges_of(rng, "documents", tokens, pool.lengths, 1)
    starts = np.concatenate([[0], np.cumsum(tokens)])
    ranges[starts[0]:starts[1]] = [[50, 50]]
    ranges[starts[2]:starts[3]] = [[6, 2 ** 31 - 1]]
    ranges[starts[3]:starts[4]] = [[-2 ** 31, -5]]
    out, lse = run(rng, pool, tokens, hq=4, ranges=ranges, cap=9.0, gated=True, word=status)
    empty = np.r_[starts[0]:starts[1], starts[2]:starts[4]]
    assert bool((out[empty] == 0).all()) and bool(torch.isneginf(lse[empty]).all())
    ranges[:] = [[3, 3]]
    run(rng, pool, tokens, hq=4, ranges=ranges, word=status)
    run(rng, pool, tokens, hq=4, ranges=ranges, sinks=2, slopes=slopes_of(4), word=status)     # but for the sinks


@pytest.mark.parametrize("act,out_dtype", [(np.float32, torch.float16), (np.float16, torch.float32), (np.float32, torch.float32)])
@pytest.mark.parametrize("d,mode", [(128, 3), (256, 0), (128, 0)])
def test_types(cuda, status, act, out_dtype, d, mode):
    rng = np.random.default_rng(d + mode)
    pool = po.Pool(rng, [50, 300, 33], d=d, heads=2, page=16, mode=mode, qblock=32)
    for tokens in ([20, 1, 33], [1, 1, 1]):
        ranges = ranges_of(rng, "prefix", tokens, pool.lengths, 1)
        run(rng, pool, tokens, hq=8, act=act, out_dtype=out_dtype, gated=True, cap=15.0, ranges=ranges, word=status)
        run(rng, pool, tokens, hq=8, act=act, out_dtype=out_dtype, slopes=slopes_of(8), ranges=ranges, word=status)


@pytest.mark.parametrize("d,heads,hq,mode", [(128, 2, 8, 3), (256, 1, 6, 0)])
def test_long_chunks_split_and_merge(cuda, status, d, heads, hq, mode):
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [4000, 700, 2500], d=d, heads=heads, page=64, mode=mode, qblock=32)
    tokens = [70, 150, 1]
    run(rng, pool, tokens, hq=hq, gated=True, q_std=2.5, cap=20.0, word=status)
    run(rng, pool, tokens, hq=hq, slopes=slopes_of(hq), window=900, sinks=4, word=status)
    run(rng, pool, tokens, hq=hq, ranges=ranges_of(rng, "prefix", tokens, pool.lengths, 1), cap=20.0, word=status)
    run(rng, pool, tokens, hq=hq, ranges=ranges_of(rng, "any", tokens, pool.lengths, 1), sinks=100, word=status)


@pytest.mark.parametrize("d,heads,hq,mode,qblock", [(128, 2, 8, 3, 32), (256, 1, 6, 0, 32), (256, 2, 16, 3, 256)])
def test_long_single_tokens_split_and_merge(cuda, status, d, heads, hq, mode, qblock):
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [9000, 700, 2500, 5], d=d, heads=heads, page=64, mode=mode, qblock=qblock)
    tokens = [1, 1, 1, 1]
    run(rng, pool, tokens, hq=hq, gated=True, q_std=2.5, cap=20.0, word=status)
    run(rng, pool, tokens, hq=hq, slopes=slopes_of(hq), window=900, sinks=4, word=status)
    ranges = np.array([[8000, 8700], [100, 700], [0, 2500], [2, 3], [7, 7]], np.int32)
    run(rng, pool, tokens, hq=hq, ranges=ranges, sinks=17, cap=20.0, slopes=slopes_of(hq), word=status)


@pytest.mark.parametrize("mode,qblock", [(3, 32), (0, 128), (1, 32)])
def test_many_documents_in_a_chunk(cuda, status, mode, qblock):
    """More row tiles than a block lays out at a time, documents that end inside tiles, a common head; a chunk that begins inside a document."""
    rng = np.random.default_rng(mode)
    lengths, tokens = [1500, 3, 900], [1400, 1, 900]
    pool = po.Pool(rng, lengths, d=128, heads=8, page=16, mode=mode, qblock=qblock)
    rows = []
    for n, length in zip(tokens, lengths):
        i = np.arange(length - n, length)
        edges = np.unique(np.concatenate([[0], rng.integers(0, length, 20)]))
        rows.append(np.stack([edges[np.searchsorted(edges, i, side="right") - 1], i + 1], 1))
    run(rng, pool, tokens, hq=32, ranges=np.concatenate(rows + [np.zeros((1, 2))]).astype(np.int32), sinks=40, pad_rows=1, cap=30.0 if mode == 3 else 0.0, word=status)


@pytest.mark.parametrize("cap", [1e-6, 0.01, 1e6])
@pytest.mark.parametrize("tokens", [[20, 33], [1, 1]])
def test_caps_far_from_the_scores(cuda, status, cap, tokens):
    """Scores that are all the cap or none near it: +cap and -cap hundreds of scores away, and a cap that changes nothing."""
    rng = np.random.default_rng(5)
    pool = po.Pool(rng, [100, 260], d=128, heads=2, page=16, mode=0, qblock=128)
    if cap < 1e6:
        run(rng, pool, tokens, hq=4, cap=cap, q_std=30.0, word=status)
        return
    # one rounding of a cap of a million is a sixteenth: tanh(x) / x is 1 to 2^-40 for these, and the polynomial's error is relative to x
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens)
    q = (1.5 * rng.standard_normal((batch.total_tokens, 4, 128))).astype(np.float16)
    got = []
    for scoring in (paged.PagedScoring(cap=cap), None):
        out = torch.zeros(q.shape, device="cuda")
        paged.launch_paged_attention(view, batch, dev(q), out, query_heads=4, scale=0.09, workspace=paged.paged_workspace(view, batch, 4, scoring=scoring), scoring=scoring)
        got.append(out)
    # scores of up to 10, off by 2^-22 of themselves more
    assert float((got[0] - got[1]).abs().max()) <= 2.0 ** -10 * float(got[1].abs().max())


@pytest.mark.parametrize("cap", [1.0, 6.0, 25.0, 400.0])
@pytest.mark.parametrize("d,kind", [(128, None), (128, "documents"), (256, "prefix")])
def test_caps_with_a_bias_over_tiles(cuda, status, cap, d, kind):
    """Scores past the cap, up to it, up to half of it and far below, each with a bias by distance, in tiles that are seen whole and in part."""
    rng = np.random.default_rng(23)
    tokens = [150, 70, 1]
    pool = po.Pool(rng, [400, 70, 333], d=d, heads=2, page=16, mode=0, qblock=d)
    ranges = None if kind is None else ranges_of(rng, kind, tokens, pool.lengths, 1)
    run(rng, pool, tokens, hq=8, ranges=ranges, cap=cap, slopes=slopes_of(8), q_std=2.0, word=status)


def test_infinite_and_nan_queries_stay_in_their_rows(cuda, status):
    rng = np.random.default_rng(6)
    pool = po.Pool(rng, [90, 40], d=128, heads=2, page=16, mode=0, qblock=128)
    view = pool.upload()
    for tokens in ([30, 1], [1, 1]):
        batch, starts = po.batch_of(pool, tokens)
        q = dev((1.5 * rng.standard_normal((batch.total_tokens, 4, 128))).astype(np.float16))
        scoring = paged.PagedScoring(cap=10.0, slopes=dev(slopes_of(4)), ranges=dev(ranges_of(rng, "documents", tokens, pool.lengths)))
        ws = paged.paged_workspace(view, batch, 4, scoring=scoring)
        clean, out = (torch.zeros(q.shape, dtype=torch.float16, device="cuda") for _ in range(2))
        paged.launch_paged_attention(view, batch, q, clean, query_heads=4, scale=0.09, workspace=ws, scoring=scoring)
        q[0, 1, 5] = float("nan")
        paged.launch_paged_attention(view, batch, q, out, query_heads=4, scale=0.09, workspace=ws, scoring=scoring)
        assert bool(out[0, 1].isnan().all())
        out[0, 1] = clean[0, 1]
        assert torch.equal(out, clean)
    assert int(status) == 0


def test_nothing_asked_for_is_plain_attention(cuda, status):
    """A scoring of nothing gives the same bits; so do ranges that say what a token sees anyway, but for the order of the pieces."""
    rng = np.random.default_rng(7)
    pool = po.Pool(rng, [300, 70, 40], d=128, heads=2, page=32, mode=3, qblock=32)
    view = pool.upload()
    for tokens in ([90, 1, 40], [1, 1, 1]):
        batch, starts = po.batch_of(pool, tokens)
        q = dev((1.5 * rng.standard_normal((batch.total_tokens, 8, 128))).astype(np.float16))
        ranges = np.concatenate([np.stack([np.zeros(n, int), np.arange(length - n, length) + 1], 1) for n, length in zip(tokens, pool.lengths)]).astype(np.int32)
        got = []
        for scoring in (None, paged.PagedScoring(), paged.PagedScoring(ranges=dev(ranges))):
            out, lse = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape[:2], device="cuda")
            paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=0.09, lse=lse, scoring=scoring, workspace=paged.paged_workspace(view, batch, 8, scoring=scoring))
            got.append((out, lse))
        assert all(torch.equal(a, b) for a, b in zip(got[0], got[1]))
        assert all(float((a - b).abs().max()) <= 2.0 ** -10 * float(a.abs().max()) for a, b in zip(got[0], got[2]))
    assert int(status) == 0


def test_bad_pages_bounds_and_padding(cuda, status):
    """A page outside the pool reads as zeros; lengths above the bounds are cut; sequences without tokens."""
    rng = np.random.default_rng(8)
    pool = po.Pool(rng, [100, 64, 30], d=128, heads=2, page=16, mode=0, qblock=128)
    for tokens in ([50, 1, 0], [1, 1, 0]):
        view = pool.upload()
        batch, starts = po.batch_of(pool, tokens, pad_rows=2)
        q = (1.5 * rng.standard_normal((batch.total_tokens, 4, 128))).astype(np.float16)
        ranges = ranges_of(rng, "prefix", tokens, pool.lengths, 2)
        scoring = paged.PagedScoring(cap=20.0, slopes=dev(slopes_of(4)), ranges=dev(ranges))
        ws = paged.paged_workspace(view, batch, 4, scoring=scoring)
        kept = pool.table[0, 2], pool.k.copy(), pool.v.copy()
        pool.table_dev[0, 2] = pool.pages + 3
        pool.k[kept[0]] = pool.v[kept[0]] = 0
        out = torch.full(q.shape, 5.0, dtype=torch.float16, device="cuda")
        paged.launch_paged_attention(view, batch, dev(q), out, query_heads=4, scale=128 ** -0.5, workspace=ws, scoring=scoring)
        want, _, bound, _ = so.attention(pool, q, starts, 128 ** -0.5, cap=20.0, slopes=slopes_of(4), ranges=ranges)
        n = int(starts[-1])
        assert (np.abs(out.cpu().numpy().astype(np.float64)[:n] - want[:n]) <= bound[:n]).all() and bool((out[n:] == 5).all())
        assert int(status) == paged.STATUS_BAD_PAGE
        status.zero_()
        pool.k, pool.v = kept[1], kept[2]
        pool.upload()
        batch, starts = po.batch_of(pool, tokens, pad_rows=2)
        batch.tensors[2].copy_(po.ints([100, 5000, 30]))            # above the bound
        paged.launch_paged_attention(view, batch, dev(q), out, query_heads=4, scale=0.09, workspace=ws, scoring=scoring)
        assert int(status) == paged.STATUS_BAD_BOUND | paged.STATUS_BAD_PAGE      # cut to the bound, where its table has no pages
        status.zero_()


def test_starts_that_do_not_ascend_cost_results_only(cuda, status):
    """Two sequences with the same rows: their row tiles share places in the workspace, and there may be more of them than it has room for.  The call ends, says so, and the next one is right."""
    rng = np.random.default_rng(12)
    pool = po.Pool(rng, [400] * 9, d=128, heads=1, page=16, mode=0, qblock=128)
    view = pool.upload()
    for hq in (1, 8):
        batch, _ = po.batch_of(pool, [400] * 9, starts=[0] + [400, 0] * 4 + [400], total_tokens=400, max_tokens=400)
        q = dev((1.5 * rng.standard_normal((400, hq, 128))).astype(np.float16))
        ranges = dev(np.stack([rng.integers(0, 400, 400), np.full(400, 400)], 1).astype(np.int32))
        scoring = paged.PagedScoring(ranges=ranges, cap=20.0)
        ws = paged.paged_workspace(view, batch, hq, scoring=scoring)
        guard = torch.full((ws.numel() + 4096,), 77, dtype=torch.uint8, device="cuda")
        out = torch.zeros(q.shape, dtype=torch.float16, device="cuda")
        paged.launch_paged_attention(view, batch, q, out, query_heads=hq, scale=0.09, workspace=guard[:ws.numel()], scoring=scoring)
        assert int(status) & paged.STATUS_BAD_BOUND and bool((guard[ws.numel():] == 77).all())
        status.zero_()
        run(rng, pool, [40, 1, 0, 17, 400, 1, 1, 9, 64], hq=hq, ranges=ranges_of(rng, "documents", [40, 1, 0, 17, 400, 1, 1, 9, 64], pool.lengths, 1), cap=20.0, poison=False, word=status)


def test_captured_replayed_and_two_graphs_over_one_workspace(cuda, status):
    """A step captured once replays with other ranges, slopes and lengths; two graphs that share a workspace, one after the other."""
    rng = np.random.default_rng(9)
    pool = po.Pool(rng, [300, 90, 40], d=128, heads=2, page=16, mode=3, qblock=32)
    view = pool.upload()
    steps = []
    for tokens in ([40, 1, 5], [1, 1, 1]):
        batch, starts = po.batch_of(pool, tokens)
        q = (1.5 * rng.standard_normal((batch.total_tokens, 8, 128))).astype(np.float16)
        ranges, slopes = dev(ranges_of(rng, "documents", tokens, pool.lengths)), dev(slopes_of(8))
        steps.append(dict(tokens=tokens, batch=batch, starts=starts, q=q, q_dev=dev(q), ranges=ranges, slopes=slopes, out=torch.zeros(q.shape, dtype=torch.float16, device="cuda"),
                          scoring=paged.PagedScoring(cap=12.0, slopes=slopes, ranges=ranges)))
    ws = torch.empty(max(paged.paged_workspace(view, s["batch"], 8, scoring=s["scoring"], sinks=3).numel() for s in steps), dtype=torch.uint8, device="cuda")
    for s in steps:
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            paged.launch_paged_attention(view, s["batch"], s["q_dev"], s["out"], query_heads=8, scale=128 ** -0.5, workspace=ws, scoring=s["scoring"], sinks=3)
    lengths = list(pool.lengths)
    for turn in range(3):
        for s in steps:
            pool.lengths = lengths if turn == 0 else [250, 64, 39]
            s["batch"].tensors[2].copy_(po.ints(pool.lengths))
            ranges, slopes = ranges_of(rng, ("documents", "prefix", "any")[turn], s["tokens"], pool.lengths), slopes_of(8) * (turn + 1)
            s["ranges"].copy_(dev(ranges))
            s["slopes"].copy_(dev(slopes))
            s["graph"].replay()
            want, _, bound, _ = so.attention(pool, s["q"], s["starts"], 128 ** -0.5, cap=12.0, slopes=slopes, ranges=ranges, sinks=3)
            assert (np.abs(s["out"].cpu().numpy().astype(np.float64) - want) <= bound).all()
    pool.lengths = lengths
    assert int(status) == 0


def test_a_stream_of_its_own_and_two_calls_at_once(cuda, status):
    rng = np.random.default_rng(10)
    pool = po.Pool(rng, [500, 90, 40], d=128, heads=2, page=16, mode=3, qblock=32)
    view = pool.upload()
    streams, calls = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for stream, tokens in zip(streams, ([200, 1, 40], [1, 1, 1])):
        batch, starts = po.batch_of(pool, tokens)
        q = (1.5 * rng.standard_normal((batch.total_tokens, 8, 128))).astype(np.float16)
        ranges = ranges_of(rng, "prefix", tokens, pool.lengths)
        scoring = paged.PagedScoring(cap=12.0, ranges=dev(ranges))
        calls.append((stream, batch, starts, q, dev(q), ranges, scoring, paged.paged_workspace(view, batch, 8, scoring=scoring), torch.zeros(q.shape, dtype=torch.float16, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(3):
        for stream, batch, _, _, q, _, scoring, ws, out in calls:
            paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=128 ** -0.5, workspace=ws, scoring=scoring, stream=stream)
    torch.cuda.synchronize()
    for _, _, starts, q, _, ranges, _, _, out in calls:
        want, _, bound, _ = so.attention(pool, q, starts, 128 ** -0.5, cap=12.0, ranges=ranges)
        assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()
    assert int(status) == 0


@pytest.mark.parametrize("d,mode", [(128, 0), (256, 3)])
def test_many_sequences_with_ranges(cuda, status, d, mode):
    """More sequences than the blocks that look at their ranges, most of a token and some of a chunk, empty ones among them."""
    rng = np.random.default_rng(d)
    lengths = [int(x) for x in rng.integers(1, 60, 700)]
    tokens = [0 if i % 11 == 3 else 1 for i in range(700)]
    for i in range(5, 700, 37):
        lengths[i] = tokens[i] = int(rng.integers(9, 60))
    pool = po.Pool(rng, lengths, d=d, heads=1, page=16, mode=mode, qblock=32)
    run(rng, pool, tokens, hq=4, ranges=ranges_of(rng, "documents", tokens, lengths, 1), sinks=2, cap=20.0, word=status)
    run(rng, pool, tokens, hq=4, ranges=ranges_of(rng, "any", tokens, lengths, 1), slopes=slopes_of(4), word=status)


@pytest.mark.parametrize("scores", [dict(slopes=True), dict(kind="prefix"), dict(slopes=True, kind="documents")])
@pytest.mark.parametrize("d", [128, 256])
def test_statistics_of_fp32_queries_over_fp16_keys(cuda, status, scores, d):
    """Without a cap they are as good as those of fp16 queries: what the queries' rounding to fp16 does to them is put back, up to its square and the rounding of the mean keys."""
    rng = np.random.default_rng(d + len(scores))
    pool = po.Pool(rng, [300, 70, 40], d=d, heads=2, page=32, mode=0, qblock=32)
    view, tokens, hq = pool.upload(), [90, 9, 40], 8
    batch, starts = po.batch_of(pool, tokens)
    q = (1.5 * rng.standard_normal((batch.total_tokens, hq, d))).astype(np.float32)
    slopes = slopes_of(hq) if "slopes" in scores else None
    ranges = ranges_of(rng, scores["kind"], tokens, pool.lengths) if "kind" in scores else None
    scoring = paged.PagedScoring(slopes=None if slopes is None else dev(slopes), ranges=None if ranges is None else dev(ranges))
    out, lse = torch.zeros(q.shape, device="cuda"), torch.zeros(q.shape[:2], device="cuda")
    paged.launch_paged_attention(view, batch, dev(q), out, query_heads=hq, scale=d ** -0.5, lse=lse, scoring=scoring, workspace=paged.paged_workspace(view, batch, hq, scoring=scoring))
    exact = q.astype(np.float16).astype(np.float64)
    want, want_lse, _, _ = so.attention(pool, q, starts, d ** -0.5, slopes=slopes, ranges=ranges)
    _, _, _, limit = so.attention(pool, q.astype(np.float16), starts, d ** -0.5, slopes=slopes, ranges=ranges)      # of queries that need no rounding
    left = np.abs(q - exact)
    most = max(np.abs(pool.rows(s, h, 0)).max() for s in range(3) for h in range(2))
    moved = left.sum(-1) * most * d ** -0.5                        # the most that the rounding moves a score by
    # the square of it (the weights' own change times the scores'), and the mean key's rounding to fp16, with the weights' and the sum's: 2^-10 of what it corrects
    assert (np.abs(lse.cpu().numpy() - want_lse) <= limit + 2 * moved ** 2 + moved * 2.0 ** -10).all()
    assert int(status) == 0


def test_tensors_that_are_refused(cuda):
    rng = np.random.default_rng(11)
    pool = po.Pool(rng, [30], d=128, heads=1, page=16, mode=0, qblock=128)
    view = pool.upload()
    batch, _ = po.batch_of(pool, [4])
    q, out = torch.zeros(4, 4, 128, dtype=torch.float16, device="cuda"), torch.zeros(4, 4, 128, dtype=torch.float16, device="cuda")
    go = lambda scoring, ws=None: paged.launch_paged_attention(view, batch, q, out, query_heads=4, scale=0.1, scoring=scoring,
                                                               workspace=paged.paged_workspace(view, batch, 4, scoring=scoring) if ws is None else ws)
    f, r = torch.zeros(4, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    go(paged.PagedScoring(cap=3.0, slopes=f, ranges=r))
    for bad in (dict(slopes=f.half()), dict(slopes=f[None]), dict(ranges=r.long()), dict(ranges=r[:, :1]), dict(ranges=r.flatten()), dict(ranges=r.t()), dict(slopes=torch.zeros(8, device="cuda")[::2])):
        with pytest.raises(ValueError):
            paged.PagedScoring(**bad)
    for bad in (dict(slopes=f[:3].clone()), dict(ranges=r[:3].clone())):
        with pytest.raises(ValueError):
            go(paged.PagedScoring(**bad))
    for bad in (dict(cap=-1.0), dict(cap=float("nan")), dict(cap=1e-9)):
        with pytest.raises(paged._lib.B200KvError):
            go(paged.PagedScoring(**bad))
    with pytest.raises(paged._lib.B200KvError):
        go(paged.PagedScoring(ranges=r), paged.paged_workspace(view, batch, 4))       # no room for the ranges' bounds

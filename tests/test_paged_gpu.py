"""The operators over a paged cache against plain implementations in 64 bits, through the public entry points."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import kv, paged

pytestmark = pytest.mark.gpu

MODES = [(0, 32), (3, 32), (3, None), (1, 32), (2, None), (2, 32), (1, None)]      # (quant mode, qblock; None = head_dim)


@pytest.fixture
def status():
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    kv.set_status_word(word)
    yield word
    kv.set_status_word(None)


# ---- store and load ---------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("d,heads,page,dtype,rope,norm", [(128, 8, 16, np.float16, 1, False), (256, 4, 64, np.float32, 2, True), (128, 3, 256, np.float32, 1, True),
                                                          (256, 6, 32, np.float16, 0, False)])
def test_store_writes_the_rows_of_the_contiguous_store(cuda, status, mode, qblock, d, heads, page, dtype, rope, norm):
    rng = np.random.default_rng(1000 * mode + d + page)
    tokens, lengths = [3, 0, 1, 40, 17], [19, 5, 1, 40, 300]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=page, mode=mode, qblock=qblock or d)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=2)
    total = batch.total_tokens
    k, v = (to_dev(rng.standard_normal((total, heads * d)).astype(dtype)) for _ in range(2))
    w = to_dev((1 + 0.1 * rng.standard_normal(d)).astype(np.float32)) if norm else None
    before = [None if p is None else p.clone() for p in pool.dev]
    for shift in (0, 1234):
        positions = None
        if shift:
            positions = po.ints([lengths[s] - tokens[s] + t + shift + 7 * s for s in range(5) for t in range(tokens[s])] + [0, 0])
        paged.launch_paged_store(view, batch, k, v, w, rope_mode=kv.RopeMode(rope), positions=positions)
        expected = [None if p is None else p.clone() for p in before]
        for s, n in enumerate(tokens):
            if n == 0:
                continue
            base = lengths[s] - n + (shift + 7 * s if shift else 0)
            st = kv.AttentionLayerKvCacheStorage(base + n, kv.KvCacheQuantMode(mode), kv_heads=heads, head_dim=d, qblock=qblock or d)
            kv.launch_kv_store_quant(st.view(), k[starts[s]:starts[s] + n], v[starts[s]:starts[s] + n], w, n, base, rope_mode=kv.RopeMode(rope))
            planes = [st.key_cache if st.key_cache is not None else st.key_cache_q8, st.key_scales, st.value_cache if st.value_cache is not None else st.value_cache_q8, st.value_scales]
            for e, plane in zip(expected, planes):
                if e is None:
                    continue
                for t in range(n):
                    pg, slot = pool.place(s, lengths[s] - n + t)
                    e[pg, :, slot] = plane[:, base + t]
        for got, e in zip(pool.dev, expected):
            assert got is None or torch.equal(got, e)
        key, value = (torch.full((total, heads, d), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
        paged.launch_paged_load(view, batch, key, value)
        pool.k, pool.ks, pool.v, pool.vs = (None if p is None else p.cpu().numpy() for p in pool.dev)
        for s, n in enumerate(tokens):
            for h in range(heads):
                for side, got in ((0, key), (1, value)):
                    want = pool.rows(s, h, side)[lengths[s] - n:].astype(np.float16)
                    assert np.array_equal(got[starts[s]:starts[s + 1], h].cpu().numpy(), want)
        assert bool((key[-2:] == 7).all() and (value[-2:] == 7).all())
        for p, e in zip(pool.dev, before):
            if p is not None:
                p.copy_(e)
    alone = torch.zeros(total, heads, d, dtype=torch.float16, device="cuda")
    paged.launch_paged_store(view, batch, k, v, w, rope_mode=kv.RopeMode(rope), positions=positions)
    paged.launch_paged_load(view, batch, None, alone)
    assert torch.equal(alone[:-2], value[:-2])
    assert int(status) == 0


def test_store_skips_pages_outside_the_pool_and_says_so(cuda, status):
    rng = np.random.default_rng(5)
    pool = po.Pool(rng, [40, 33], d=128, heads=2, page=16, mode=3, qblock=32)
    good = pool.table.copy()
    pool.table[0, 2] = pool.pages
    pool.table[1, 2] = -1
    view = pool.upload()
    batch, _ = po.batch_of(pool, [12, 3])
    k, v = (torch.randn(15, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) for _ in range(2))
    before = [p.clone() for p in pool.dev]
    paged.launch_paged_store(view, batch, k, v, None)
    changed = (pool.dev[0] != before[0]).any(-1).any(1).cpu().numpy()      # [page][slot]
    allowed = np.zeros_like(changed)
    allowed[good[0, 1], 12:] = True                                       # positions 28 .. 31; 32 .. 39 and 32 lie on the bad pages
    allowed[good[1, 1], 14:] = True                                       # positions 30, 31
    assert not (changed & ~allowed).any() and changed.any()
    assert int(status) == paged.STATUS_BAD_PAGE
    status.zero_()
    out = torch.full((15, 2, 128), 3.0, dtype=torch.float16, device="cuda")
    paged.launch_paged_load(view, batch, out, None)
    assert bool((out[4:12] == 0).all()) and bool((out[:4] != 0).any()) and int(status) == paged.STATUS_BAD_PAGE


# ---- attention --------------------------------------------------------------------------------------------------------------------------


def run_attention(rng, pool, tokens, *, hq, act=np.float16, out_dtype=torch.float16, window=0, sinks=0, gated=False, pad_rows=1, q_std=1.5, stale=True, **bounds):
    view = pool.upload()
    if stale:      # what lies past a length may be anything
        for s, n in enumerate(pool.lengths):
            if n % pool.page:
                pg = int(pool.table[s, n // pool.page])
                for p in pool.dev:
                    if p is not None and p.dtype == torch.float16:
                        p[pg, :, n % pool.page:] = float("nan")
    batch, starts = po.batch_of(pool, tokens, pad_rows=pad_rows, **bounds)
    total, d = batch.total_tokens, pool.d
    q = (q_std * rng.standard_normal((total, hq, d))).astype(act)
    gate = rng.standard_normal((total, hq, d)).astype(np.float32) if gated else None
    out = torch.full((total, hq, d), 5.0, dtype=out_dtype, device="cuda")
    lse = torch.full((total, hq), 5.0, device="cuda")
    ws = paged.paged_workspace(view, batch, hq, window=window, sinks=sinks)
    ws.fill_(255)
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=hq, scale=d ** -0.5, window=window, sinks=sinks,
                                 gate=None if gate is None else to_dev(gate), lse=lse, workspace=ws)
    want, want_lse, bound = po.attention(pool, q, starts, d ** -0.5, window, sinks, gate)
    n = int(starts[-1])
    got = out.cpu().numpy().astype(np.float64)
    assert (got[n:] == 5.0).all() and bool((lse[n:] == 5.0).all())
    off = np.abs(got[:n] - want[:n])
    worst = np.unravel_index(np.argmax(off - bound[:n]), off.shape)
    assert (off <= bound[:n]).all(), (worst, got[:n][worst], want[:n][worst], bound[:n][worst], float((off > bound[:n]).mean()))
    got_lse = lse[:n].cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isneginf(got_lse), np.isneginf(want_lse[:n]))
    fine = np.isfinite(want_lse[:n])
    # the statistics: scores as in the output's bound, the sum of weights that are rounded once
    rounded = po.HALF_STEP * ((pool.mode in (1, 3)) + (act == np.float32))
    most = max((np.abs(pool.rows(s, h, 0)).sum(-1).max() if pool.lengths[s] else 0.0) for s in range(len(tokens)) for h in range(pool.heads))
    limit = most * np.abs(q.astype(np.float64)).max() * d ** -0.5 * (rounded + 2.0 ** -20) + po.HALF_STEP + 2.0 ** -20 * np.abs(want_lse[:n][fine]).max(initial=1.0)
    assert (np.abs(got_lse[fine] - want_lse[:n][fine]) <= limit).all()
    return out, lse


@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("d,heads,hq,page", [(128, 2, 8, 16), (256, 2, 12, 64), (128, 3, 3, 256), (256, 1, 8, 32)])
def test_attention_of_ragged_chunks(cuda, status, mode, qblock, d, heads, hq, page):
    rng = np.random.default_rng(100 * mode + d + hq)
    pool = po.Pool(rng, [40, 9, 1, 130, 65, 7, 200], d=d, heads=heads, page=page, mode=mode, qblock=qblock or d)
    run_attention(rng, pool, [40, 0, 1, 2, 5, 7, 33], hq=hq, gated=hq == 12)
    assert int(status) == 0


@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("d,heads,hq,page", [(128, 8, 32, 64), (256, 4, 24, 16), (128, 2, 2, 128), (256, 3, 24, 32), (128, 1, 7, 16)])
def test_attention_of_single_tokens(cuda, status, mode, qblock, d, heads, hq, page):
    rng = np.random.default_rng(100 * mode + d + hq)
    pool = po.Pool(rng, [1, 2, 15, 16, 17, 127, 128, 129, 500, 1000], d=d, heads=heads, page=page, mode=mode, qblock=qblock or d)
    run_attention(rng, pool, [1, 1, 1, 1, 1, 0, 1, 1, 1, 1], hq=hq, gated=hq == 24)
    assert int(status) == 0


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (50, 0), (64, 1), (100, 70), (129, 17), (1000, 5), (5, 300)])
@pytest.mark.parametrize("d,mode,hq", [(128, 0, 8), (256, 3, 4)])
def test_attention_with_a_window_and_sinks(cuda, status, window, sinks, d, mode, hq):
    rng = np.random.default_rng(window + sinks + d)
    lengths, tokens = [300, 70, 40, 130, 260], [90, 1, 40, 3, 1]
    pool = po.Pool(rng, lengths, d=d, heads=2, page=32, mode=mode, qblock=32)
    for s, length in enumerate(lengths):       # what no token of the sequence sees is large: a position too many shows
        seen = np.zeros(length, bool)
        for t in range(tokens[s]):
            seen |= po.mask_of(length - tokens[s] + t, length, window, sinks)
        for j in np.flatnonzero(~seen):
            pg, slot = pool.place(s, j)
            if mode == 0:
                pool.v[pg, :, slot] = 3.0e4
            else:
                pool.vs[pg, :, slot] = 200.0
    run_attention(rng, pool, tokens, hq=hq, window=window, sinks=sinks)
    assert int(status) == 0


@pytest.mark.parametrize("act,out_dtype", [(np.float32, torch.float16), (np.float16, torch.float32), (np.float32, torch.float32)])
@pytest.mark.parametrize("d,mode", [(128, 3), (256, 0)])
def test_attention_types(cuda, act, out_dtype, d, mode):
    rng = np.random.default_rng(d + mode)
    pool = po.Pool(rng, [50, 300, 33], d=d, heads=2, page=16, mode=mode, qblock=32)
    run_attention(rng, pool, [20, 1, 33], hq=8, act=act, out_dtype=out_dtype, gated=True)
    run_attention(rng, pool, [1, 1, 1], hq=8, act=act, out_dtype=out_dtype, gated=True)


@pytest.mark.parametrize("d,heads,hq,mode", [(128, 2, 8, 3), (256, 1, 6, 0)])
def test_attention_of_long_chunks_splits_and_merges(cuda, status, d, heads, hq, mode):
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [4000, 700, 2500], d=d, heads=heads, page=64, mode=mode, qblock=32)
    run_attention(rng, pool, [70, 150, 1], hq=hq, gated=True, q_std=2.5)
    run_attention(rng, pool, [70, 150, 1], hq=hq, window=900, sinks=4)
    assert int(status) == 0


@pytest.mark.parametrize("d,heads,hq,mode,qblock", [(128, 2, 8, 3, 32), (256, 1, 6, 0, 32), (256, 2, 16, 3, 256)])
def test_attention_of_long_single_tokens_splits_and_merges(cuda, status, d, heads, hq, mode, qblock):
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [9000, 700, 2500, 5], d=d, heads=heads, page=64, mode=mode, qblock=qblock)
    run_attention(rng, pool, [1, 1, 1, 1], hq=hq, gated=True, q_std=2.5)
    run_attention(rng, pool, [1, 1, 1, 1], hq=hq, window=900, sinks=4)
    assert int(status) == 0


@pytest.mark.parametrize("d,heads,hq,mode,qblock", [(128, 8, 32, 3, 32), (128, 8, 32, 0, 32), (256, 4, 24, 3, 32), (256, 4, 16, 0, 32), (256, 4, 24, 3, 256), (128, 8, 64, 1, 32)])
def test_attention_of_many_sequences_whose_pieces_cross_from_one_to_the_next(cuda, status, d, heads, hq, mode, qblock):
    """Pieces of a dozen tiles and more, most of them with the ends of two or three kv heads."""
    rng = np.random.default_rng(d + mode)
    lengths = [int(x) for x in rng.integers(1, 3500, 36)]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=64, mode=mode, qblock=qblock)
    tokens = [1] * 36
    tokens[7] = tokens[20] = 0
    run_attention(rng, pool, tokens, hq=hq, stale=False)
    if hq == 32:
        tokens[5] = 2       # eight rows: the other kernel for all
        run_attention(rng, pool, tokens, hq=hq, stale=False)
    assert int(status) == 0


def test_attention_where_scores_reach_far(cuda):
    """Scores of several hundred, the largest last or first."""
    rng = np.random.default_rng(3)
    for order in (1, -1):
        pool = po.Pool(rng, [400, 257], d=128, heads=1, page=16, mode=0, qblock=128)
        q = rng.standard_normal(128)
        for s, length in enumerate(pool.lengths):
            for i, j in enumerate(range(length)[::order]):
                pg, slot = pool.place(s, j)
                pool.k[pg, 0, slot] = (q * (i / length) * 3).astype(np.float16)
        view = pool.upload()
        for tokens in ([30, 257], [1, 1]):
            batch, starts = po.batch_of(pool, tokens)
            qs = np.broadcast_to((q * 4).astype(np.float16), (batch.total_tokens, 4, 128)).copy()
            out = torch.zeros(batch.total_tokens, 4, 128, device="cuda")
            paged.launch_paged_attention(view, batch, to_dev(qs), out, query_heads=4, scale=1.0, workspace=paged.paged_workspace(view, batch, 4))
            want, _, bound = po.attention(pool, qs, starts, 1.0)
            # scores of 1500 in fp32: 2^-24 of them per rounding of score and reference
            slack = np.abs(qs.astype(np.float64)).sum() * 0 + 4 * 1600 * 2.0 ** -24 * np.abs(pool.v.astype(np.float64)).max()
            assert (np.abs(out.cpu().numpy() - want) <= bound + slack).all()


def test_values_a_single_token_does_not_see_never_count(cuda):
    """Infinities and NaN under the mask: between the sinks and the window, and behind the length."""
    rng = np.random.default_rng(11)
    for d in (128, 256):
        pool = po.Pool(rng, [200, 90, 333], d=d, heads=2, page=16, mode=0, qblock=32)
        window, sinks = 37, 3
        for s, length in enumerate(pool.lengths):
            m = po.mask_of(length - 1, length, window, sinks)
            for n, j in enumerate(np.flatnonzero(~m)):
                pg, slot = pool.place(s, j)
                pool.k[pg, :, slot], pool.v[pg, :, slot] = [(np.nan, np.nan), (np.inf, -np.inf), (-np.inf, np.inf)][n % 3]
        clean = po.Pool.__new__(po.Pool)
        clean.__dict__.update(pool.__dict__)
        clean.k, clean.v = np.nan_to_num(pool.k, nan=0, posinf=0, neginf=0), np.nan_to_num(pool.v, nan=0, posinf=0, neginf=0)
        view = pool.upload()
        batch, starts = po.batch_of(pool, [1, 1, 1])
        q = rng.standard_normal((3, 8, d)).astype(np.float16)
        out = torch.zeros(3, 8, d, dtype=torch.float16, device="cuda")
        paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=8, scale=d ** -0.5, window=window, sinks=sinks,
                                     workspace=paged.paged_workspace(view, batch, 8, window=window, sinks=sinks))
        want, _, bound = po.attention(clean, q, starts, d ** -0.5, window, sinks)
        assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()


def test_bad_pages_read_as_zeros_and_bounds_cut(cuda, status):
    rng = np.random.default_rng(2)
    for tokens in ([20, 20], [1, 1]):
        pool = po.Pool(rng, [100, 100], d=128, heads=2, page=16, mode=3, qblock=32)
        good = pool.table.copy()
        view = pool.upload()
        bad = pool.table_dev.clone()
        bad[0, 2], bad[1, 1] = 1 << 30, -5
        pool.table_dev = bad
        batch, starts = po.batch_of(pool, tokens)
        q = rng.standard_normal((sum(tokens), 4, 128)).astype(np.float16)
        out = torch.zeros(sum(tokens), 4, 128, dtype=torch.float16, device="cuda")
        ws = paged.paged_workspace(view, batch, 4)
        paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=4, scale=0.1, workspace=ws)
        for s, j in ((0, 2), (1, 1)):
            pool.vs[good[s, j]] = 0
            pool.ks[good[s, j]] = 0
        want, _, bound = po.attention(pool, q, starts, 0.1)
        assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()
        assert int(status) == paged.STATUS_BAD_PAGE
        status.zero_()
        # lengths and starts that contradict the bounds: cut, reported, nothing behind the rows touched
        pool.table_dev = torch.from_numpy(good).cuda()
        for lengths, begin in (([1000000, -3], None), ([100, 100], [0, sum(tokens) + 50, sum(tokens) + 90]), ([100, 100], [5, 3, -1])):
            batch, _ = po.batch_of(pool, tokens, starts=[0, *np.cumsum(tokens)])
            arrays = po.ints(lengths), po.ints(begin if begin is not None else [0, *np.cumsum(tokens)])
            batch.lengths, batch.query_starts = arrays[0].data_ptr(), arrays[1].data_ptr()
            guard = torch.full((sum(tokens) + 8, 4, 128), 9.0, dtype=torch.float16, device="cuda")
            paged.launch_paged_attention(view, batch, to_dev(q), guard[:sum(tokens)], query_heads=4, scale=0.1, workspace=ws)
            assert bool((guard[sum(tokens):] == 9).all()) and int(status) == paged.STATUS_BAD_BOUND
            status.zero_()


# ---- weights ----------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("mode,qblock", [(0, 32), (3, 32), (3, None), (1, 32)])
@pytest.mark.parametrize("d,heads,hq,act,window,sinks,observe", [(128, 2, 8, np.float16, 0, 0, 0), (256, 1, 6, np.float16, 40, 3, 0), (128, 3, 3, np.float32, 0, 0, 5),
                                                                 (256, 2, 16, np.float32, 100, 17, 30)])
def test_weights(cuda, status, mode, qblock, d, heads, hq, act, window, sinks, observe):
    rng = np.random.default_rng(10 * mode + d + hq)
    lengths, tokens = [300, 9, 1, 130, 257, 64], [70, 0, 1, 2, 40, 1]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=16, mode=mode, qblock=qblock or d)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=1)
    q = (1.5 * rng.standard_normal((batch.total_tokens, hq, d))).astype(act)
    _, lse, _ = po.attention(pool, q, starts, d ** -0.5, window, sinks)
    lse = np.nan_to_num(lse, nan=0.0, neginf=-np.inf).astype(np.float32)
    stride = max(lengths) + 13
    before = rng.random((len(lengths), heads, stride)).astype(np.float32) * 0.01
    w = to_dev(before)
    paged.launch_paged_weights(view, batch, to_dev(q), to_dev(lse), w, query_heads=hq, scale=d ** -0.5, window=window, sinks=sinks, observe=observe)
    added, bounds = po.weights(pool, q, lse, starts, d ** -0.5, window, sinks, observe)
    got = w.cpu().numpy()
    for s, length in enumerate(lengths):
        want = before[s, :, :length] + added[s]
        limit = bounds[s] + np.abs(want) * 2.0 ** -23
        off = np.abs(got[s, :, :length].astype(np.float64) - want)
        assert (off <= limit).all(), (s, np.unravel_index(np.argmax(off - limit), off.shape), off.max())
        assert np.array_equal(got[s, :, length:], before[s, :, length:])
    assert int(status) == 0


def test_weights_of_a_row_that_sees_nothing(cuda):
    rng = np.random.default_rng(1)
    pool = po.Pool(rng, [2, 30], d=128, heads=1, page=16, mode=0, qblock=128)
    view = pool.upload()
    batch, starts = po.batch_of(pool, [5, 2])       # three tokens lie before the cache's beginning
    q = rng.standard_normal((7, 2, 128)).astype(np.float16)
    out, lse = torch.full((7, 2, 128), 4.0, device="cuda"), torch.zeros(7, 2, device="cuda")
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=2, scale=0.1, lse=lse, workspace=paged.paged_workspace(view, batch, 2))
    assert bool((out[:3] == 0).all()) and bool(torch.isneginf(lse[:3]).all()) and bool(torch.isfinite(lse[3:]).all())
    w = torch.zeros(2, 1, 30, device="cuda")
    paged.launch_paged_weights(view, batch, to_dev(q), lse, w, query_heads=2, scale=0.1)
    assert abs(float(w[0].sum()) - 4) < 1e-4 and abs(float(w[1].sum()) - 4) < 1e-4      # two tokens of two heads each


# ---- eviction ---------------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("mode,qblock", MODES)
@pytest.mark.parametrize("d,heads,page,keep,sinks,recent", [(128, 2, 16, 50, 4, 10), (256, 3, 64, 128, 0, 0), (128, 1, 256, 7, 3, 4), (256, 2, 32, 1, 0, 0), (128, 2, 16, 1200, 2, 300)])
def test_evict(cuda, status, in_place, mode, qblock, d, heads, page, keep, sinks, recent):
    rng = np.random.default_rng(keep + d + mode)
    lengths = [300, 0, keep, keep + 1, 3000, 17]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=page, mode=mode, qblock=qblock or d, spare=2 + 6 * -(-keep // page))
    view = pool.upload()
    batch, _ = po.batch_of(pool, [0] * 6, pad_rows=1)
    stride = max(lengths) + 5
    w = rng.standard_normal((6, heads, stride)).astype(np.float32)
    w[:, :, ::3] = np.round(w[:, :, ::3] * 4) / 4              # many ties
    w[:, 0, 5:200:7] = 0.0
    w[:, 0, 6:200:7] = -0.0
    w[0, 0, 20:40] = np.nan
    w[4, 0, 100:110] = [np.inf, -np.inf, 1e-41, 2e-41, -1e-41, 3e38, -3e38, 0.0, -0.0, np.nan]
    need = -(-keep // page)
    if in_place:
        target = batch.tensors[0]
        if target.shape[1] * page < keep:
            pytest.skip("the sequences' own table is no larger")
    else:
        target = torch.from_numpy(pool.spare[:6 * need].reshape(6, need).astype(np.int32)).cuda()
    kept = torch.full((6, heads, keep), 99, dtype=torch.int32, device="cuda")
    new_w, new_len = torch.full((6, heads, keep), 99.0, device="cuda"), torch.full((6,), 99, dtype=torch.int32, device="cuda")
    before = [None if p is None else p.cpu().numpy().copy() for p in pool.dev]
    paged.launch_paged_evict(view, batch, target, to_dev(w), keep=keep, sinks=sinks, recent=recent, kept=kept, new_lengths=new_len, new_weights=new_w)
    expected = [None if p is None else p.copy() for p in before]
    tt = target.cpu().numpy()
    for s, length in enumerate(lengths):
        for h in range(heads):
            want = po.evict(w[s, h], length, keep, sinks, recent)
            got = kept[s, h].cpu().numpy()
            assert np.array_equal(got[:len(want)], want) and (got[len(want):] == -1).all(), (s, h)
            np.testing.assert_array_equal(new_w[s, h].cpu().numpy(), np.concatenate([w[s, h, want], np.zeros(keep - len(want), np.float32)]))
            for r, j in enumerate(want):
                pg, slot = pool.place(s, j)
                for e, b in zip(expected, before):
                    if e is not None:
                        e[tt[s, r // page], h, r % page] = b[pg, h, slot]
    assert new_len.tolist() == [min(n, keep) for n in lengths]
    for p, e in zip(pool.dev, expected):
        if p is not None:
            assert np.array_equal(p.cpu().numpy().view(np.int8), e.view(np.int8))
    assert int(status) == 0


def test_evict_a_long_sequence(cuda):
    rng = np.random.default_rng(8)
    pool = po.Pool(rng, [40000, 12345], d=128, heads=2, page=128, mode=3, qblock=32)
    view = pool.upload()
    w = np.abs(rng.standard_normal((2, 2, 40000))).astype(np.float32)
    w[1] = np.round(w[1] * 8) / 8
    for keep, sinks, recent in ((4096, 4, 1000), (20000, 0, 1)):
        batch, _ = po.batch_of(pool, [0, 0], pad_rows=1)
        kept, new_len = torch.zeros(2, 2, keep, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        planes = [p.clone() for p in pool.dev]
        paged.launch_paged_evict(view, batch, pool.table_dev, to_dev(w), keep=keep, sinks=sinks, recent=recent, kept=kept, new_lengths=new_len)
        for s, length in enumerate(pool.lengths):
            for h in range(2):
                want = po.evict(w[s, h], length, keep, sinks, recent)
                assert np.array_equal(kept[s, h, :len(want)].cpu().numpy(), want)
                r = torch.arange(len(want), device="cuda")
                j = torch.from_numpy(want).cuda()
                t = pool.table_dev[s].long()
                for p, b in zip(pool.dev, planes):
                    assert torch.equal(p[t[r // 128], h, r % 128], b[t[j // 128], h, j % 128])
        for p, b in zip(pool.dev, planes):
            p.copy_(b)


# ---- together ---------------------------------------------------------------------------------------------------------------------------


def test_a_sequence_lives_store_attend_weigh_evict_and_goes_on(cuda, status):
    """Prompts stored in two pieces, attention and weights of each, eviction in place, then tokens at positions that are no longer their places."""
    rng = np.random.default_rng(21)
    d, heads, hq, page, keep = 128, 2, 8, 16, 60
    lengths = [150, 80]
    pool = po.Pool(rng, [0, 0], d=d, heads=heads, page=page, mode=3, qblock=32, capacity=200)
    view = pool.upload()
    scale = d ** -0.5
    account = torch.zeros(2, heads, 200, device="cuda")
    expected = np.zeros((2, heads, 200))

    def step(tokens, positions=None):
        batch, starts = po.batch_of(pool, tokens, max_length=200, total_length=400)
        n = sum(tokens)
        k, v = (to_dev(rng.standard_normal((n, heads * d)).astype(np.float16)) for _ in range(2))
        q = (1.5 * rng.standard_normal((n, hq, d))).astype(np.float16)
        paged.launch_paged_store(view, batch, k, v, None, rope_mode=kv.RopeMode.NEOX_FULL, positions=positions)
        out, lse = torch.zeros(n, hq, d, dtype=torch.float16, device="cuda"), torch.zeros(n, hq, device="cuda")
        paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=hq, scale=scale, lse=lse, workspace=paged.paged_workspace(view, batch, hq))
        paged.launch_paged_weights(view, batch, to_dev(q), lse, account, query_heads=hq, scale=scale)
        pool.k, pool.ks, pool.v, pool.vs = (p.cpu().numpy() for p in pool.dev)
        want, _, bound = po.attention(pool, q, starts, scale)
        assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()
        added, limit = po.weights(pool, q, lse.cpu().numpy(), starts, scale)
        for s, length in enumerate(pool.lengths):
            got = account[s, :, :length].cpu().numpy()
            expected[s, :, :length] += added[s]
            assert (np.abs(got - expected[s, :, :length]) <= 4 * limit[s] + 2.0 ** -20 * np.abs(got)).all()
            expected[s, :, :length] = got
        return batch

    pool.lengths = [100, 50]
    step([100, 50])
    pool.lengths = lengths
    batch = step([50, 30])
    kept, new_len = torch.zeros(2, heads, keep, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    new_w = torch.zeros(2, heads, keep, device="cuda")
    paged.launch_paged_evict(view, batch, pool.table_dev, account, keep=keep, sinks=2, recent=20, kept=kept, new_lengths=new_len, new_weights=new_w)
    for s in range(2):
        for h in range(heads):
            assert np.array_equal(kept[s, h].cpu().numpy(), po.evict(account[s, h].cpu().numpy(), lengths[s], keep, 2, 20))
    account.zero_()
    account[:, :, :keep] = new_w
    expected[:] = account.cpu().numpy()
    assert new_len.tolist() == [keep, keep]
    pool.lengths = [keep + 1, keep + 2]
    step([1, 2], positions=po.ints([150, 80, 81]))
    pool.lengths = [keep + 2, keep + 3]
    step([1, 1], positions=po.ints([151, 82]))
    assert int(status) == 0


@pytest.mark.parametrize("tokens", [[1, 1, 1], [40, 1, 9]])
def test_a_captured_step_replays_with_what_the_arrays_hold(cuda, status, tokens):
    """One graph, other lengths, starts and pages on each replay; a second graph with a workspace of its own replayed in between."""
    rng = np.random.default_rng(31)
    d, heads, hq = 128, 2, 8
    pool = po.Pool(rng, [300, 400, 200], d=d, heads=heads, page=32, mode=3, qblock=32)
    view = pool.upload()
    scale = d ** -0.5
    starts_dev, lengths_dev, n = po.ints([0, 0, 0, 0]), po.ints([0, 0, 0]), sum(tokens)
    batch = paged.PagedBatch(pool.table_dev, starts_dev, lengths_dev, total_tokens=n, max_tokens=max(tokens), max_length=400, total_length=900)
    q = to_dev(rng.standard_normal((n, hq, d)).astype(np.float16))
    stream = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        out, lse, w = torch.zeros(n, hq, d, dtype=torch.float16, device="cuda"), torch.zeros(n, hq, device="cuda"), torch.zeros(3, heads, 400, device="cuda")
        ws = paged.paged_workspace(view, batch, hq, window=150, sinks=4)
        stream.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            paged.launch_paged_attention(view, batch, q, out, query_heads=hq, scale=scale, window=150, sinks=4, lse=lse, workspace=ws)
            paged.launch_paged_weights(view, batch, q, lse, w, query_heads=hq, scale=scale, window=150, sinks=4)
        graphs.append((g, out, lse, w, ws))
    full = pool.lengths
    for lengths in (full, [45, 77, 10], [300, 0, 33]):
        toks = [min(t, l) for t, l in zip(tokens, lengths)]
        starts = np.concatenate([[0], np.cumsum(toks)])
        starts_dev.copy_(po.ints(starts))
        lengths_dev.copy_(po.ints(lengths))
        pool.lengths = lengths
        want, _, bound = po.attention(pool, q.cpu().numpy(), starts, scale, 150, 4)
        for g, out, lse, w, _ in graphs:
            w.zero_()
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, out, lse, w, _ in graphs:
            m = int(starts[-1])
            assert (np.abs(out[:m].cpu().numpy().astype(np.float64) - want[:m]) <= bound[:m]).all()
            added, limit = po.weights(pool, q.cpu().numpy(), lse.cpu().numpy(), starts, scale, 150, 4)
            for s in range(3):
                assert (np.abs(w[s, :, :lengths[s]].cpu().numpy() - added[s]) <= limit[s] + 2.0 ** -24).all()
    assert int(status) == 0


def test_calls_on_another_stream_and_under_launch_overlap(cuda):
    rng = np.random.default_rng(41)
    pool = po.Pool(rng, [200, 90], d=128, heads=2, page=16, mode=0, qblock=32)
    view = pool.upload()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    kv.set_launch_overlap(1)
    try:
        for tokens in ([1, 1], [30, 4]):
            batch, starts = po.batch_of(pool, tokens)
            n = sum(tokens)
            k, v = (torch.randn(n, 256, device="cuda").half() for _ in range(2))
            q = to_dev(rng.standard_normal((n, 8, 128)).astype(np.float16))
            out, ws = torch.zeros(n, 8, 128, dtype=torch.float16, device="cuda"), paged.paged_workspace(view, batch, 8)
            torch.cuda.synchronize()
            for _ in range(3):
                paged.launch_paged_store(view, batch, k, v, None, stream=stream)
                paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=0.1, workspace=ws, stream=stream)
            stream.synchronize()
            pool.k, pool.ks, pool.v, pool.vs = (None if p is None else p.cpu().numpy() for p in pool.dev)
            want, _, bound = po.attention(pool, q.cpu().numpy(), starts, 0.1)
            assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()
    finally:
        kv.set_launch_overlap(0)

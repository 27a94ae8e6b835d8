"""The operators over a paged cache at the edges of what their calls allow: every group of heads on both sides of the kernels' limits, hundreds of sequences,
pages that sequences share, calls side by side and replayed, lengths past what registers hold; against plain implementations in 64 bits."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import kv, paged
from test_paged_gpu import MODES, run_attention, status  # noqa: F401

pytestmark = pytest.mark.gpu


def run_weights(rng, pool, tokens, *, hq, act=np.float16, window=0, sinks=0, observe=0, extra=3):
    """Adds to random weights; entries at and past a length stay."""
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=1)
    scale = pool.d ** -0.5
    q = (1.5 * rng.standard_normal((batch.total_tokens, hq, pool.d))).astype(act)
    _, lse, _ = po.attention(pool, q, starts, scale, window, sinks)
    lse = np.nan_to_num(lse, nan=0.0, neginf=-np.inf).astype(np.float32)
    before = rng.random((len(pool.lengths), pool.heads, max(pool.lengths) + extra)).astype(np.float32) * 0.01
    w = to_dev(before)
    paged.launch_paged_weights(view, batch, to_dev(q), to_dev(lse), w, query_heads=hq, scale=scale, window=window, sinks=sinks, observe=observe)
    added, bounds = po.weights(pool, q, lse, starts, scale, window, sinks, observe)
    got = w.cpu().numpy()
    for s, length in enumerate(pool.lengths):
        want = before[s, :, :length] + added[s]
        off = np.abs(got[s, :, :length].astype(np.float64) - want)
        limit = bounds[s] + np.abs(want) * 2.0 ** -23      # the sum is rounded once more, to fp32
        assert (off <= limit).all(), (s, np.unravel_index(np.argmax(off - limit), off.shape), off.max())
        assert np.array_equal(got[s, :, length:], before[s, :, length:])
    return w


@pytest.mark.parametrize("group", range(1, 9))
@pytest.mark.parametrize("d,mode,qblock,page", [(128, 3, 32, 16), (256, 0, 256, 32), (256, 3, 256, 16), (128, 2, 128, 64)])
def test_attention_on_both_sides_of_the_few_rows(cuda, status, group, d, mode, qblock, page):
    rng = np.random.default_rng(group + d + mode)
    for tokens, lengths in ([1, 2, 3, 4, 5, 8, 9], [130, 2, 128, 129, 6, 140, 9]), ([1, 2, 1, 1], [127, 300, 1, 128]), ([0, 8 // group, 1, 0], [5, 8 // group, 257, 0]):
        pool = po.Pool(rng, lengths, d=d, heads=2, page=page, mode=mode, qblock=qblock)
        run_attention(rng, pool, tokens, hq=2 * group, window=0 if group % 2 else 100, sinks=3)
    assert int(status) == 0


@pytest.mark.parametrize("group", range(1, 9))
@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 3, 32), (128, 0, 128), (256, 0, 256), (256, 1, 256)])
def test_weights_of_few_rows(cuda, status, group, d, mode, qblock):
    rng = np.random.default_rng(7 * group + d + mode)
    pool = po.Pool(rng, [130, 2, 128, 129, 0, 300, 1], d=d, heads=2, page=16, mode=mode, qblock=qblock)
    for tokens, window, act in ([1, 1, 1, 1, 0, 1, 1], 0, np.float16), ([8 // group, 1, 0, 1, 0, 1, 1], 60, np.float32):
        run_weights(rng, pool, tokens, hq=2 * group, act=act, window=window, sinks=5 if window else 0)
    run_weights(rng, pool, [20, 2, 9, 50, 0, 70, 1], hq=2 * group, observe=8 // group)      # of long chunks, the last few tokens
    assert int(status) == 0


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 3, 32), (128, 0, 128), (256, 0, 256), (128, 3, 128), (256, 1, 256)])
@pytest.mark.parametrize("heads,group,window", [(1, 5, 0), (2, 7, 333), (3, 1, 0), (1, 8, 130)])
def test_weights_of_long_chunks(cuda, status, act, d, mode, qblock, heads, group, window):
    rng = np.random.default_rng(heads + group + d + mode)
    pool = po.Pool(rng, [700, 260, 129], d=d, heads=heads, page=32, mode=mode, qblock=qblock)
    run_weights(rng, pool, [300, 129, 64], hq=heads * group, act=act, window=window, sinks=9)
    assert int(status) == 0


@pytest.mark.parametrize("sequences", [129, 300])
@pytest.mark.parametrize("most", [1, 30])
def test_hundreds_of_sequences(cuda, status, sequences, most):
    rng = np.random.default_rng(sequences + most)
    lengths = rng.integers(0, 150, sequences)
    lengths[5], lengths[sequences - 2] = 900, 700
    tokens = np.minimum(rng.integers(0, 2, sequences) if most == 1 else np.where(rng.random(sequences) < 0.1, most, rng.integers(0, 4, sequences)), lengths)
    pool = po.Pool(rng, [int(n) for n in lengths], d=128, heads=2, page=16, mode=3, qblock=32)
    run_attention(rng, pool, [int(n) for n in tokens], hq=4)
    run_weights(rng, pool, [int(n) for n in tokens], hq=4)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens)
    total = batch.total_tokens
    key, value = (torch.zeros(total, 2, 128, dtype=torch.float16, device="cuda") for _ in range(2))
    paged.launch_paged_load(view, batch, key, value)
    for s in range(sequences):
        for side, got in ((0, key), (1, value)):
            want = np.stack([pool.rows(s, h, side)[lengths[s] - tokens[s]:] for h in range(2)], 1).astype(np.float16)
            assert np.array_equal(got[starts[s]:starts[s + 1]].cpu().numpy(), want)
    assert int(status) == 0


@pytest.mark.parametrize("tokens", [[1, 1, 1], [33, 1, 70]])
@pytest.mark.parametrize("d,mode", [(128, 3), (256, 0)])
def test_sequences_that_share_their_first_pages(cuda, status, tokens, d, mode):
    rng = np.random.default_rng(d)
    pool = po.Pool(rng, [300, 330, 260], d=d, heads=2, page=16, mode=mode, qblock=32)
    pool.table[1:, :10] = pool.table[0, :10]
    run_attention(rng, pool, tokens, hq=8)
    run_weights(rng, pool, tokens, hq=8)
    assert int(status) == 0


@pytest.mark.parametrize("tokens", [[1, 1], [40, 3]])
def test_windows_that_are_none_and_sinks_past_the_length(cuda, tokens):
    rng = np.random.default_rng(3)
    pool = po.Pool(rng, [200, 77], d=128, heads=2, page=16, mode=3, qblock=32)
    run_attention(rng, pool, tokens, hq=8, window=50, sinks=5000)
    view = pool.upload()
    batch, _ = po.batch_of(pool, tokens)
    q = to_dev(rng.standard_normal((sum(tokens), 8, 128)).astype(np.float16))
    found = []
    for window, sinks in ((0, 0), (0, 9), (200, 3), (0xffffffff, 0xffffffff)):
        out, lse, w = torch.zeros_like(q), torch.zeros(sum(tokens), 8, device="cuda"), torch.zeros(2, 2, 200, device="cuda")
        paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=0.09, window=window, sinks=sinks, lse=lse, workspace=paged.paged_workspace(view, batch, 8, window=window, sinks=sinks))
        paged.launch_paged_weights(view, batch, q, lse, w, query_heads=8, scale=0.09, window=window, sinks=sinks, observe=0 if window else 1000)
        found.append((out, lse, w))
    for other in found[1:]:
        assert all(torch.equal(a, b) for a, b in zip(found[0], other))


@pytest.mark.parametrize("tokens", [[1, 1, 1, 1], [90, 1, 30, 2]])
def test_the_same_call_gives_the_same_bits_alone_and_beside_another(cuda, tokens):
    """Two streams, each with its own workspace, pools and results."""
    rng = np.random.default_rng(sum(tokens))
    made = []
    for mode in (3, 0):
        pool = po.Pool(rng, [3000, 250, 1000, 128], d=128, heads=4, page=64, mode=mode, qblock=32)
        view = pool.upload()
        batch, _ = po.batch_of(pool, tokens)
        q = to_dev(rng.standard_normal((sum(tokens), 16, 128)).astype(np.float16))
        made.append((view, batch, q, paged.paged_workspace(view, batch, 16), torch.cuda.Stream(), pool))

    def call(view, batch, q, ws, stream, out, lse, w):
        paged.launch_paged_attention(view, batch, q, out, query_heads=16, scale=0.09, lse=lse, workspace=ws, stream=stream)
        paged.launch_paged_weights(view, batch, q, lse, w, query_heads=16, scale=0.09, stream=stream)

    results = lambda: [(torch.zeros(sum(tokens), 16, 128, device="cuda"), torch.zeros(sum(tokens), 16, device="cuda"), torch.zeros(4, 4, 3000, device="cuda")) for _ in made]
    alone = results()
    torch.cuda.synchronize()
    for m, r in zip(made, alone):
        call(*m[:5], *r)
        torch.cuda.synchronize()
    for _ in range(5):
        beside = results()
        torch.cuda.synchronize()
        for _ in range(2):
            for m, r in zip(made, beside):
                r[2].record_stream(m[4])
                with torch.cuda.stream(m[4]):
                    r[2].zero_()
                call(*m[:5], *r)
        torch.cuda.synchronize()
        for a, b in zip(alone, beside):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_graphs_replayed_in_turn_share_a_workspace(cuda):
    rng = np.random.default_rng(77)
    pool = po.Pool(rng, [2000, 300, 500], d=256, heads=2, page=32, mode=3, qblock=256)
    view = pool.upload()
    stream, made = torch.cuda.Stream(), []
    batches = [po.batch_of(pool, t) for t in ([100, 2, 1], [1, 1, 1], [1, 40, 3])]
    ws = torch.empty(max(paged.paged_workspace(view, b, 12).numel() for b, _ in batches), dtype=torch.uint8, device="cuda").fill_(255)
    stream.wait_stream(torch.cuda.current_stream())
    for batch, starts in batches:
        q = to_dev(rng.standard_normal((batch.total_tokens, 12, 256)).astype(np.float16))
        out = torch.zeros_like(q)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            paged.launch_paged_attention(view, batch, q, out, query_heads=12, scale=0.06, workspace=ws)
        made.append((graph, q, out, *po.attention(pool, q.cpu().numpy(), starts, 0.06)))     # (the graph reads q where it was)
    for _ in range(3):
        for graph, _, out, *_ in made:
            out.fill_(7.0)
            graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, _, bound in made:
            assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all()


@pytest.mark.parametrize("max_tokens", [1, 200])
def test_a_batch_in_which_nothing_is_new_leaves_everything(cuda, status, max_tokens):
    rng = np.random.default_rng(2)
    pool = po.Pool(rng, [40, 0, 200], d=128, heads=2, page=16, mode=3, qblock=32)
    view = pool.upload()
    before = [p.clone() for p in pool.dev]
    batch, _ = po.batch_of(pool, [0, 0, 0], pad_rows=300, max_tokens=max_tokens)
    q = torch.randn(300, 8, 128, device="cuda")
    out, lse, w = torch.full_like(q, 3.0), torch.full((300, 8), 3.0, device="cuda"), torch.full((3, 2, 200), 3.0, device="cuda")
    rows = torch.randn(300, 256, device="cuda")
    key = torch.full((300, 2, 128), 3.0, dtype=torch.float16, device="cuda")
    paged.launch_paged_store(view, batch, rows, rows, None)
    paged.launch_paged_load(view, batch, key, None)
    paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=0.1, lse=lse, workspace=paged.paged_workspace(view, batch, 8))
    paged.launch_paged_weights(view, batch, q, lse, w, query_heads=8, scale=0.1)
    for t in (out, lse, w, key):
        assert bool((t == 3).all())
    assert all(torch.equal(a, b) for a, b in zip(pool.dev, before)) and int(status) == 0


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("length", [131073, 140001])
def test_evict_more_positions_than_registers_hold(cuda, in_place, length):
    rng = np.random.default_rng(length)
    keep, page = 70000, 256
    need = -(-keep // page)
    pool = po.Pool(rng, [length, 200], d=128, heads=1, page=page, mode=0, qblock=128, spare=2 * need)
    view = pool.upload()
    batch, _ = po.batch_of(pool, [0, 0], pad_rows=1)
    target = pool.table_dev if in_place else torch.from_numpy(pool.spare.reshape(2, need).astype(np.int32)).cuda()
    w = rng.standard_normal((2, 1, length)).astype(np.float32)
    w[0, 0, ::2] = np.round(w[0, 0, ::2] * 64) / 64
    before = pool.dev[0].clone()
    kept, new_len = torch.zeros(2, 1, keep, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    paged.launch_paged_evict(view, batch, target, to_dev(w), keep=keep, sinks=4, recent=30000, kept=kept, new_lengths=new_len)
    want = po.evict(w[0, 0], length, keep, 4, 30000)
    assert np.array_equal(kept[0, 0].cpu().numpy(), want) and new_len.tolist() == [keep, 200]
    r, j = torch.arange(keep, device="cuda"), torch.from_numpy(want).cuda()
    to, of = target[0].long(), pool.table_dev[0].long() if not in_place else torch.from_numpy(pool.table[0]).cuda().long()
    assert torch.equal(pool.dev[0][to[r // page], 0, r % page], before[of[j // page], 0, j % page])


@pytest.mark.parametrize("page", [16, 256])
def test_one_position_one_token_one_head(cuda, status, page):
    rng = np.random.default_rng(page)
    for mode in range(4):
        pool = po.Pool(rng, [1], d=128, heads=1, page=page, mode=mode, qblock=32, spare=0)
        run_attention(rng, pool, [1], hq=1, pad_rows=0)
        w = run_weights(rng, pool, [1], hq=1, extra=0)
        view = pool.upload()
        batch, _ = po.batch_of(pool, [1])
        kept, new_len = torch.zeros(1, 1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        paged.launch_paged_evict(view, batch, batch.tensors[0], w, keep=1, kept=kept, new_lengths=new_len)
        assert kept.item() == 0 and new_len.item() == 1
    assert int(status) == 0


def test_calls_refuse_tensors_that_do_not_fit(cuda):
    rng = np.random.default_rng(1)
    pool = po.Pool(rng, [40, 30], d=128, heads=2, page=16, mode=3, qblock=32)
    view = pool.upload()
    batch, _ = po.batch_of(pool, [3, 1])
    half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    f32, i32 = lambda *s: torch.zeros(*s, device="cuda"), lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    ws = paged.paged_workspace(view, batch, 8)
    attend = lambda q=half(4, 8, 128), out=half(4, 8, 128), ws=ws, **k: paged.launch_paged_attention(view, batch, q, out, query_heads=8, scale=0.1, workspace=ws, **k)
    weigh = lambda q=half(4, 8, 128), lse=f32(4, 8), w=f32(2, 2, 40): paged.launch_paged_weights(view, batch, q, lse, w, query_heads=8, scale=0.1)
    evict = lambda table=i32(2, 1), w=f32(2, 2, 40), kept=i32(2, 2, 16), lengths=i32(2), **k: paged.launch_paged_evict(view, batch, table, w, keep=16, kept=kept, new_lengths=lengths, **k)
    for call in (lambda: paged.launch_paged_store(view, batch, half(3, 256), half(4, 256), None), lambda: paged.launch_paged_store(view, batch, half(4, 256), f32(4, 256), None),
                 lambda: paged.launch_paged_store(view, batch, half(4, 256).t(), half(4, 256), None), lambda: paged.launch_paged_store(view, batch, half(4, 256).bfloat16(), half(4, 256), None),
                 lambda: paged.launch_paged_store(view, batch, half(4, 256), half(4, 256), f32(127)), lambda: paged.launch_paged_store(view, batch, half(4, 256), half(4, 256), half(128)),
                 lambda: paged.launch_paged_store(view, batch, half(4, 256), half(4, 256), None, positions=i32(3)),
                 lambda: paged.launch_paged_store(view, batch, half(4, 256), half(4, 256), None, positions=i32(4).long()),
                 lambda: paged.launch_paged_load(view, batch, f32(4, 2, 128), None), lambda: paged.launch_paged_load(view, batch, half(3, 2, 128), None),
                 lambda: attend(q=half(3, 8, 128)), lambda: attend(out=half(3, 8, 128)), lambda: attend(gate=half(4, 8, 128)), lambda: attend(gate=f32(3, 8, 128)), lambda: attend(lse=f32(3, 8)),
                 lambda: attend(ws=f32(1 << 20)), lambda: weigh(q=half(3, 8, 128)), lambda: weigh(lse=f32(3, 8)), lambda: weigh(lse=half(4, 8)), lambda: weigh(w=f32(2, 2, 39)),
                 lambda: weigh(w=half(2, 2, 40)), lambda: evict(table=i32(2, 1).long()), lambda: evict(w=f32(2, 2, 39)), lambda: evict(kept=i32(2, 2, 15)), lambda: evict(lengths=i32(1)),
                 lambda: evict(new_weights=f32(2, 2, 15)), lambda: evict(kept=f32(2, 2, 16))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: attend(ws=ws[:-1]), lambda: attend(ws=None), lambda: attend(q=half(33, 128).view(-1)[4:4 + 4096]), lambda: evict(lengths=batch.tensors[2]),
                 lambda: evict(table=i32(2, 0)), lambda: paged.launch_paged_load(view, batch, None, None)):
        with pytest.raises((kv.B200KvError, ValueError)):
            call()
    elsewhere = pool.upload()
    elsewhere.device_index = torch.cuda.current_device() + 1
    with pytest.raises(ValueError, match="another device"):
        paged.launch_paged_load(elsewhere, batch, half(4, 2, 128), None)
    torch.cuda.synchronize()


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("d,heads,hq,window,sinks", [(128, 2, 8, 3, 0), (128, 1, 4, 19, 0), (256, 2, 12, 40, 4), (256, 1, 1, 0, 0), (128, 2, 14, 0, 0)])
def test_statistics_of_chunks_are_good_to_their_type(cuda, status, act, d, heads, hq, window, sinks):
    """Over an fp16 cache nothing but products and sums of 32 bits stands between a chunk's lse and the formula: neither rounded queries nor rounded weights."""
    rng = np.random.default_rng(d + hq + window)
    lengths, tokens = [300, 64, 900, 1, 40], [70, 64, 130, 1, 2]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=16, mode=0, qblock=d)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=3)
    total, n = batch.total_tokens, sum(tokens)
    q = (1.5 * rng.standard_normal((total, hq, d))).astype(act)
    out, lse = torch.zeros(total, hq, d, dtype=torch.float16, device="cuda"), torch.full((total, hq), 5.0, device="cuda")
    ws = paged.paged_workspace(view, batch, hq, window=window, sinks=sinks).fill_(255)
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=hq, scale=d ** -0.5, window=window, sinks=sinks, lse=lse, workspace=ws)
    _, want, _ = po.attention(pool, q, starts, d ** -0.5, window, sinks)
    got = lse.cpu().numpy().astype(np.float64)
    assert (got[n:] == 5.0).all() and int(status) == 0
    # a score: d products in fp32 and its scale, 2^-20 of the largest sum of magnitudes; exponentials of 2 units of 2^-23 each, their sums of fewer than 1024 terms half a
    # unit a step and on average half of that, 2^-17 of a sum at the most; the logarithm and its factor 2^-21 of the value.  fp32 queries: a score moves by e, at most
    # 2^-11 of the sum of magnitudes; the first order is taken out but for the mean key's rounding and its fp16 weights (2^-9 of it), the second is e^2 / 2
    most = max(np.abs(pool.rows(s, h, 0)).sum(-1).max() for s in range(5) for h in range(heads)) * np.abs(q.astype(np.float64)).max() * d ** -0.5
    magnitude = max((np.abs(pool.rows(s, h, 0)) @ np.abs(q[starts[s]:starts[s + 1], h * (hq // heads):(h + 1) * (hq // heads)].reshape(-1, d).astype(np.float64)).T).max()
                    for s in range(5) for h in range(heads)) * d ** -0.5
    assert magnitude <= most
    e = 2.0 ** -11 * magnitude if act == np.float32 else 0.0
    limit = 2.0 ** -20 * magnitude + 2.0 ** -17 + 2.0 ** -21 * np.abs(want[:n]) + e * 2.0 ** -9 + e * e / 2
    off = np.abs(got[:n] - want[:n])
    assert (off <= limit).all(), (off.max(), limit.max())
    # as a whole, in the 2-norm, to 1e-5 (roundings do not lie at their limits all at once)
    assert np.linalg.norm(off) <= 1e-5 * np.linalg.norm(want[:n])


@pytest.mark.parametrize("chunk", [1, 20])
def test_the_most_sequences(cuda, status, chunk):
    rng = np.random.default_rng(chunk)
    lengths = [int(n) for n in rng.integers(0, 4, 8192)]
    lengths[4000] = lengths[8191] = 40
    tokens = [min(n, 1) if s % 2 else 0 for s, n in enumerate(lengths)]
    tokens[4000] = tokens[8191] = chunk
    pool = po.Pool(rng, lengths, d=128, heads=1, page=16, mode=3, qblock=32)
    run_attention(rng, pool, tokens, hq=2)
    run_weights(rng, pool, tokens, hq=2)
    view = pool.upload()
    batch, _ = po.batch_of(pool, tokens)
    kept, new_len = torch.zeros(8192, 1, 2, dtype=torch.int32, device="cuda"), torch.zeros(8192, dtype=torch.int32, device="cuda")
    w = torch.rand(8192, 1, 40, device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    paged.launch_paged_evict(view, batch, batch.tensors[0], w, keep=2, sinks=1, kept=kept, new_lengths=new_len)
    host, found = w.cpu().numpy(), kept.cpu().numpy()
    for s, n in enumerate(lengths):
        want = po.evict(host[s, 0], n, 2, 1, 0)
        assert np.array_equal(found[s, 0, :len(want)], want) and (found[s, 0, len(want):] == -1).all()
    assert new_len.tolist() == [min(n, 2) for n in lengths] and int(status) == 0

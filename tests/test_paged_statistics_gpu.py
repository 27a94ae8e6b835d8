"""The statistics (lse) of attention over int8 keys, held to what the arithmetic of the kernel that a sequence takes can cost them."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import paged
from test_paged_gpu import status  # noqa: F401

pytestmark = pytest.mark.gpu

U = po.HALF_STEP      # fp16: half a step, 2^-11 of the value


def call(pool, view, batch, q, hq, *, window=0, sinks=0):
    out, lse = torch.zeros(*q.shape, dtype=torch.float16, device="cuda"), torch.full(q.shape[:2], 5.0, device="cuda")
    ws = paged.paged_workspace(view, batch, hq, window=window, sinks=sinks).fill_(255)
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=hq, scale=pool.d ** -0.5, window=window, sinks=sinks, lse=lse, workspace=ws)
    return out, lse


def rows_of(pool, q, starts, window, sinks):
    """Of every row that sees something: (token, head, its query, its keys, its weights, its lse)."""
    group = q.shape[1] // pool.heads
    for s, length in enumerate(pool.lengths):
        n = int(starts[s + 1] - starts[s])
        for h in range(pool.heads):
            k = pool.rows(s, h, 0)
            for t in range(n):
                m = po.mask_of(length - n + t, length, window, sinks)
                for e in range(h * group, (h + 1) * group):
                    row = q[starts[s] + t, e].astype(np.float64)
                    x = k[m] @ row * pool.d ** -0.5
                    p = np.exp(x - x.max())
                    yield starts[s] + t, e, row, k[m], p / p.sum(), x.max() + np.log(p.sum())


def own_arithmetic(pool, row, keys, lse):
    """What 32 bits cost: the sums of a score's products, at most 2^-20 of their magnitudes (eight blocks' sums, each exact, and their scales); exponentials of 2 units
    of 2^-23 and sums of fewer than 1100 of them, a thread's every 128th, 2^-19 together; maximum, logarithm and factor 2^-21 of the value."""
    return 2.0 ** -20 * (np.abs(keys) @ np.abs(row)).max() * pool.d ** -0.5 + 2.0 ** -19 + 2.0 ** -21 * abs(lse)


@pytest.mark.parametrize("group", range(1, 9))
@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 3, 32), (256, 3, 256), (128, 1, 128), (256, 1, 32)])
@pytest.mark.parametrize("act,outlier", [(np.float16, 1.0), (np.float32, 20.0)])
def test_of_few_rows(cuda, status, group, d, mode, qblock, act, outlier):
    """Queries are whole numbers of 24 bits against int8 keys: off by at most half of amax / (127 * 2^16), 2^-23 of amax with its own rounding, in every element.  One
    channel `outlier` times as large as the others makes that as large beside them."""
    rng = np.random.default_rng(100 * group + d + mode)
    lengths = [1, 2, 17, 128, 129, 300, 1030, 1]
    pool = po.Pool(rng, lengths, d=d, heads=2, page=16, mode=mode, qblock=qblock)
    view = pool.upload()
    for tokens in ([1, 1, 1, 1, 1, 8 // group, 1, 1], [1, 0, 1, 1, 1, 1, 1, 1]):
        of_tokens(rng, pool, view, tokens, group, act, outlier, status)


def of_tokens(rng, pool, view, tokens, group, act, outlier, word):
    d = pool.d
    batch, starts = po.batch_of(pool, tokens, pad_rows=1)
    q = (1.5 * rng.standard_normal((batch.total_tokens, 2 * group, d)))
    q[:, :, 5] *= outlier
    q = q.astype(act)
    window, sinks = (0, 0) if group % 2 else (200, 3)
    _, lse = call(pool, view, batch, q, 2 * group, window=window, sinks=sinks)
    got = lse.cpu().numpy().astype(np.float64)
    off, wants = [], []
    for token, head, row, keys, _, want in rows_of(pool, q, starts, window, sinks):
        limit = own_arithmetic(pool, row, keys, want) + np.abs(keys).sum(-1).max() * np.abs(row).max() * d ** -0.5 * 2.0 ** -23
        off.append(abs(got[token, head] - want))
        wants.append(want)
        assert off[-1] <= limit, (token, head, off[-1], limit)
    # as a whole (roundings do not lie at their limits all at once)
    assert np.linalg.norm(off) <= 4e-6 * np.linalg.norm(wants)
    assert int(word) == 0 and bool((lse[-1] == 5.0).all())


@pytest.mark.parametrize("group", [3, 5, 6, 8])
@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 3, 32), (256, 3, 256), (128, 1, 128), (256, 1, 32)])
@pytest.mark.parametrize("act,outlier", [(np.float16, 1.0), (np.float16, 20.0), (np.float32, 20.0)])
def test_the_output_alone_of_few_rows(cuda, status, group, d, mode, qblock, act, outlier):
    """Where neither statistics nor an fp32 output are asked for, queries of five to eight rows may be whole numbers of 16 bits: off by at most half of amax / (127 * 2^8), 2^-16.9 of
    amax with its own rounding, in every element; the weights move with the scores.  With statistics the output is that of 24 bits."""
    rng = np.random.default_rng(100 * group + d + mode)
    lengths = [1, 2, 17, 129, 300, 1030]
    pool = po.Pool(rng, lengths, d=d, heads=2, page=16, mode=mode, qblock=qblock)
    view = pool.upload()
    tokens = [1, 1, 1, 1, 8 // group, 1]
    batch, starts = po.batch_of(pool, tokens)
    q = 1.5 * rng.standard_normal((batch.total_tokens, 2 * group, d))
    q[:, :, 5] *= outlier
    q = q.astype(act)
    want, _, bound = po.attention(pool, q, starts, d ** -0.5)
    more = np.zeros_like(bound)
    for token, head, row, keys, p, _ in rows_of(pool, q, starts, 0, 0):
        s = int(np.searchsorted(starts, token, side="right")) - 1
        moved = np.abs(keys).sum(-1).max() * np.abs(row).max() * d ** -0.5 * 2.0 ** -16.9
        more[token, head] = np.expm1(2 * moved) * (p @ np.abs(pool.rows(s, head // group, 1)[:len(keys)]))
    out = torch.zeros(*q.shape, dtype=torch.float16, device="cuda")
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=2 * group, scale=d ** -0.5, workspace=paged.paged_workspace(view, batch, 2 * group).fill_(255))
    assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound + more).all()
    out, _ = call(pool, view, batch, q, 2 * group)
    assert (np.abs(out.cpu().numpy().astype(np.float64) - want) <= bound).all() and int(status) == 0


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("d,heads,hq,mode,qblock,window,sinks", [(128, 2, 8, 3, 32, 0, 0), (256, 1, 6, 3, 32, 0, 0), (256, 1, 6, 1, 256, 130, 4), (128, 2, 2, 3, 128, 19, 0), (128, 1, 7, 1, 32, 0, 0)])
def test_of_chunks(cuda, status, act, d, heads, hq, mode, qblock, window, sinks):
    """The chunk kernel reads int8 rows as fp16, each element off by at most U of itself, and fp32 queries likewise.  A row's lse moves by the mean over its weights
    of what its scores move: a sum of terms e_i a_i of |e_i| <= U, as good as independent, which is beyond 6 U sqrt(sum a_i^2) with a
    probability of 2 exp(-18); the second order is half of the square of the largest move of a score."""
    rng = np.random.default_rng(d + hq + mode)
    lengths, tokens = [300, 64, 900, 40, 12], [70, 64, 130, 11, 12]
    pool = po.Pool(rng, lengths, d=d, heads=heads, page=16, mode=mode, qblock=qblock)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=3)
    q = (1.5 * rng.standard_normal((batch.total_tokens, hq, d))).astype(act)
    _, lse = call(pool, view, batch, q, hq, window=window, sinks=sinks)
    got = lse.cpu().numpy().astype(np.float64)
    for token, head, row, keys, p, want in rows_of(pool, q, starts, window, sinks):
        terms = (keys * row * d ** -0.5) ** 2
        moved = np.sqrt((p ** 2) @ terms.sum(-1))
        most = (np.abs(keys) @ np.abs(row)).max() * d ** -0.5 * U
        if act == np.float32:
            moved = moved + np.sqrt((((p @ keys) * row * d ** -0.5) ** 2).sum())
            most *= 2
        limit = own_arithmetic(pool, row, keys, want) + 2.0 ** -17 + 6 * U * moved + most ** 2 / 2
        assert abs(got[token, head] - want) <= limit, (token, head, got[token, head], want, limit)
    assert int(status) == 0 and bool((lse[-3:] == 5.0).all())


@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 1, 256), (256, 3, 32)])
def test_of_chunks_with_fp32_queries_over_int8_keys_take_one_pass(cuda, d, mode, qblock):
    """Over int8 keys, which the copy rounds, the statistics are those of the queries as the kernel multiplies them: a second pass would take out no more than the
    smaller half of what the roundings cost."""
    rng = np.random.default_rng(d + mode)
    pool = po.Pool(rng, [300, 64], d=d, heads=2, page=16, mode=mode, qblock=qblock)
    view = pool.upload()
    batch, _ = po.batch_of(pool, [70, 64])
    q = (1.5 * rng.standard_normal((134, 8, d))).astype(np.float32)
    (_, lse), (_, rounded) = call(pool, view, batch, q, 8), call(pool, view, batch, q.astype(np.float16), 8)
    assert torch.equal(lse, rounded)

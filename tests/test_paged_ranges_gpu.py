"""Weights of queries, and over keys, past what fp16 holds: those of the formula, whichever kernel a sequence takes."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import paged
from test_paged_gpu import status  # noqa: F401

pytestmark = pytest.mark.gpu


def weigh(pool, q, tokens, scale, *, window=0, sinks=0, observe=0):
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens, pad_rows=1)
    _, lse, _ = po.attention(pool, q, starts, scale, window, sinks)
    lse = np.nan_to_num(lse, nan=0.0, neginf=-np.inf).astype(np.float32)
    w = torch.zeros(len(tokens), pool.heads, max(pool.lengths), device="cuda")
    paged.launch_paged_weights(view, batch, to_dev(q), to_dev(lse), w, query_heads=q.shape[1], scale=scale, window=window, sinks=sinks, observe=observe)
    added, bounds = po.weights(pool, q, lse, starts, scale, window, sinks, observe)
    got = w.cpu().numpy()
    for s, length in enumerate(pool.lengths):
        off = np.abs(got[s, :, :length].astype(np.float64) - added[s])
        limit = bounds[s] + np.abs(added[s]) * 2.0 ** -23 + 2.0 ** -126      # and a weight below the normal numbers is none
        assert (off <= limit).all(), (s, np.unravel_index(np.argmax(off - limit), off.shape), off.max(), np.isnan(got[s]).sum())


@pytest.mark.parametrize("tokens,observe", [([1, 1, 1], 0), ([90, 1, 40], 0), ([90, 65, 40], 3)])
@pytest.mark.parametrize("d,mode,qblock,heads,group", [(128, 3, 32, 2, 4), (256, 3, 32, 1, 6), (128, 0, 128, 2, 7), (256, 1, 256, 1, 1), (256, 0, 256, 1, 3)])
def test_weights_of_fp32_queries_of_any_size(cuda, status, tokens, observe, d, mode, qblock, heads, group):
    """Rows of 1e5 beside rows of 1 and of 1e-6; scores are of ordinary size by their scale, or as good as zero."""
    rng = np.random.default_rng(d + mode + group)
    pool = po.Pool(rng, [300, 129, 64], d=d, heads=heads, page=16, mode=mode, qblock=qblock)
    total = sum(tokens) + 1
    q = rng.standard_normal((total, heads * group, d)) * rng.choice([1.0e5, 1.0e5, 1.0, 1.0e-6], (total, heads * group, 1))
    q[0, 0, 3] = 1.0e5
    weigh(pool, q.astype(np.float32), tokens, 1.0e-5 * d ** -0.5, window=0 if group % 2 else 70, sinks=3, observe=observe)
    assert int(status) == 0


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("tokens,observe", [([1, 1, 1], 0), ([90, 1, 40], 0), ([90, 65, 40], 3)])
@pytest.mark.parametrize("d,heads,group", [(128, 2, 4), (256, 1, 6), (256, 2, 1)])
def test_weights_over_keys_of_any_size(cuda, status, act, tokens, observe, d, heads, group):
    """Block scales of up to 6e4 (an int8 128 of them is 8e6), down to the least that fp16 holds, beside ordinary ones, in one row and in rows of their own."""
    rng = np.random.default_rng(d + group)
    pool = po.Pool(rng, [300, 129, 64], d=d, heads=heads, page=16, mode=3, qblock=32)
    shape = pool.ks.shape
    pool.ks = np.where(rng.random(shape) < 0.1, np.float16(6.0e4), np.where(rng.random(shape) < 0.1, np.float16(6.0e-8), pool.ks)).astype(np.float16)
    pool.ks[::3] = (rng.choice([600.0, 3.0e-5], pool.ks[::3].shape[:3] + (1,)) * (1 + rng.random(pool.ks[::3].shape))).astype(np.float16)
    total = sum(tokens) + 1
    weigh(pool, rng.standard_normal((total, heads * group, d)).astype(act), tokens, 1.0e-7, window=0 if group > 1 else 70, sinks=3, observe=observe)
    assert int(status) == 0


@pytest.mark.parametrize("d,mode,qblock,heads,group", [(128, 3, 32, 2, 4), (256, 3, 32, 1, 6), (128, 0, 128, 2, 7), (256, 1, 256, 1, 1), (256, 2, 32, 1, 3)])
def test_attention_of_tokens_with_queries_and_scales_of_any_size(cuda, status, d, mode, qblock, heads, group):
    """fp32 queries of 1e5 beside ones of 1 and 1e-6; scales of up to 6e4 beside ordinary ones.  The scores are of ordinary size by their scale."""
    rng = np.random.default_rng(d + mode + group)
    pool = po.Pool(rng, [300, 129, 64, 1], d=d, heads=heads, page=16, mode=mode, qblock=qblock)
    for scales in (pool.ks, pool.vs):
        if scales is not None:
            scales[rng.random(scales.shape) < 0.05] = np.float16(6.0e4)
    view = pool.upload()
    batch, starts = po.batch_of(pool, [1, 1, 1, 1])
    q = (rng.standard_normal((4, heads * group, d)) * rng.choice([1.0e5, 1.0e5, 1.0, 1.0e-6], (4, heads * group, 1))).astype(np.float32)
    scale = 1.0e-5 * d ** -0.5 * (1.0 if pool.ks is None else 1.0e-6)
    out, lse = torch.zeros(*q.shape, device="cuda"), torch.zeros(*q.shape[:2], device="cuda")
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=heads * group, scale=scale, lse=lse, workspace=paged.paged_workspace(view, batch, heads * group))
    want, want_lse, bound = po.attention(pool, q, starts, scale)
    got = out.cpu().numpy().astype(np.float64)
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()
    assert np.allclose(lse.cpu().numpy(), want_lse, rtol=2.0 ** -18, atol=2.0 ** -17) and int(status) == 0

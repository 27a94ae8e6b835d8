"""A NaN in a query over a paged cache, whichever kernel its sequence takes."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import paged
from test_paged_gpu import status  # noqa: F401

pytestmark = pytest.mark.gpu


def attend(view, batch, q, hq, scale):
    out, lse = torch.zeros(*q.shape, device="cuda"), torch.zeros(*q.shape[:2], device="cuda")
    paged.launch_paged_attention(view, batch, to_dev(q), out, query_heads=hq, scale=scale, lse=lse, workspace=paged.paged_workspace(view, batch, hq))
    return out, lse


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("group", [1, 4, 6])
@pytest.mark.parametrize("d,mode,qblock", [(128, 3, 32), (256, 3, 256), (256, 1, 32), (128, 0, 128), (256, 2, 256)])
@pytest.mark.parametrize("tokens", [[1, 1, 1, 1], [1, 30, 2, 1]])
def test_a_nan_in_a_query_is_a_nan_in_its_row_and_in_no_other(cuda, status, act, group, d, mode, qblock, tokens):
    rng = np.random.default_rng(group + d + mode)
    pool = po.Pool(rng, [1, 300, 2000, 129], d=d, heads=2, page=16, mode=mode, qblock=qblock)
    view = pool.upload()
    batch, starts = po.batch_of(pool, tokens)
    hq, total = 2 * group, sum(tokens)
    clean = rng.standard_normal((total, hq, d)).astype(act)
    q, nan = clean.copy(), np.zeros((total, hq), bool)
    for token, head, dim in [(0, 0, 3), (int(starts[2]), hq - 1, d - 1), (int(starts[3]), hq // 2, 0)] + ([(int(starts[1]) + 7, 1, 65)] if tokens[1] > 1 else []):
        q[token, head, dim], nan[token, head] = np.nan, True
    (out, lse), (out0, lse0) = attend(view, batch, q, hq, d ** -0.5), attend(view, batch, clean, hq, d ** -0.5)
    bad = torch.from_numpy(nan).cuda()
    assert bool(torch.isnan(out[bad]).all()) and bool(torch.isnan(lse[bad]).all())
    assert torch.equal(out[~bad], out0[~bad]) and torch.equal(lse[~bad], lse0[~bad])
    # the account: a position that the row sees, of its kv head
    w, w0 = (torch.full((4, 2, 2000), 0.5, device="cuda") for _ in range(2))
    paged.launch_paged_weights(view, batch, to_dev(q), lse0, w, query_heads=hq, scale=d ** -0.5)
    paged.launch_paged_weights(view, batch, to_dev(clean), lse0, w0, query_heads=hq, scale=d ** -0.5)
    expected = torch.zeros(4, 2, 2000, dtype=torch.bool, device="cuda")
    for s, length in enumerate(pool.lengths):
        for t in range(tokens[s]):
            for head in range(hq):
                if nan[starts[s] + t, head]:
                    expected[s, head // group, :length - tokens[s] + t + 1] = True
    assert torch.equal(torch.isnan(w), expected) and torch.equal(w[~expected], w0[~expected])
    assert int(status) == 0


@pytest.mark.parametrize("act", [np.float16, np.float32])
@pytest.mark.parametrize("d,mode,heads,hq,length", [(128, 0, 8, 64, 700), (256, 3, 8, 48, 500), (128, 3, 8, 64, 60)])
def test_a_nan_in_a_chunk_whose_row_tiles_are_whole(cuda, status, act, d, mode, heads, hq, length):
    """More row tiles than multiprocessors, or too few positions to divide: a block writes its rows and their statistics itself."""
    rng = np.random.default_rng(d + length)
    pool = po.Pool(rng, [length], d=d, heads=heads, page=64, mode=mode, qblock=d)
    view = pool.upload()
    batch, _ = po.batch_of(pool, [length])
    clean = rng.standard_normal((length, hq, d)).astype(act)
    q = clean.copy()
    rows = [(0, 0), (length // 2, 3), (length - 1, hq - 1)]
    for token, head in rows:
        q[token, head, token % d] = np.nan
    (out, lse), (out0, lse0) = attend(view, batch, q, hq, d ** -0.5), attend(view, batch, clean, hq, d ** -0.5)
    bad = torch.zeros(length, hq, dtype=torch.bool, device="cuda")
    for token, head in rows:
        bad[token, head] = True
    assert bool(torch.isnan(out[bad]).all()) and bool(torch.isnan(lse[bad]).all()), lse[bad]
    assert torch.equal(out[~bad], out0[~bad]) and torch.equal(lse[~bad], lse0[~bad]) and int(status) == 0

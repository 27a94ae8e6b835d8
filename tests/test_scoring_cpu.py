"""What attention with a cap, a bias or ranges refuses, and its workspace; no GPU needed."""
import ctypes as C

import pytest
import torch

from miinfer_b200 import paged
from miinfer_b200._lib import PagedScoring, lib
from test_paged_cpu import DEVICE, INVALID, OK, RANGE, UNSUPPORTED, WORKSPACE, attend, batch_of, no_gpu, size, view_of


def scored(v, b, scoring=None, q=4096, q_dtype=0, gate=None, out=8192 * 16, out_dtype=0, lse=None, query_heads=8, scale=0.1, window=0, sinks=0, workspace=1 << 20, room=1 << 40, **k):
    s = PagedScoring(**{**dict(cap=30.0, slopes=1 << 25, ranges=1 << 26), **k}) if scoring is None else scoring
    return lib.b200kv_paged_attn_scored(C.byref(v), C.byref(b), C.byref(s), q, q_dtype, gate, out, out_dtype, lse, query_heads, scale, window, sinks, workspace, room, None)


def room(v, b, heads=8, window=0, sinks=0, **k):
    s = PagedScoring(**{**dict(cap=30.0, slopes=1 << 25, ranges=1 << 26), **k})
    return lib.b200kv_paged_attn_scored_workspace_bytes(C.byref(v), C.byref(b), C.byref(s), heads, window, sinks)


@no_gpu
@pytest.mark.parametrize("change", [{}, dict(cap=0.0), dict(slopes=None), dict(ranges=None), dict(cap=0.0, slopes=None, ranges=None), dict(window=20, sinks=3), dict(cap=1e-6), dict(cap=1e6)])
def test_calls_that_are_right_end_at_the_missing_device(change):
    assert scored(view_of(), batch_of(), **change) == DEVICE
    assert scored(view_of(), batch_of(total_tokens=3, max_tokens=1), **change) == DEVICE


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(cap=-1.0)), (INVALID, dict(cap=float("nan"))), (INVALID, dict(cap=float("inf"))), (UNSUPPORTED, dict(cap=1e-7)), (UNSUPPORTED, dict(cap=2e6)),
    (INVALID, dict(slopes=(1 << 25) + 2)), (INVALID, dict(ranges=(1 << 26) + 4)), (INVALID, dict(q=None)), (INVALID, dict(out=None)), (INVALID, dict(scale=0.0)), (INVALID, dict(query_heads=7)),
    (UNSUPPORTED, dict(query_heads=18)), (INVALID, dict(lse=2)), (WORKSPACE, dict(workspace=None)), (WORKSPACE, dict(room=room(view_of(), batch_of()) - 1)),
    (INVALID, dict(slopes=8192 * 16)), (INVALID, dict(ranges=8192 * 16 + 9 * 8 * 128 * 2 - 8)), (INVALID, dict(ranges=8192 * 16 - 8 * 9 + 8)), (INVALID, dict(lse=1 << 26)), (INVALID, dict(lse=(1 << 25) + 28)),
])
def test_arguments_that_are_refused(status, change):
    assert scored(view_of(), batch_of(), **change) == status


@pytest.mark.parametrize("status,view,batch", [(UNSUPPORTED, dict(head_dim=64), {}), (INVALID, dict(value_q8=None), {}), (RANGE, {}, dict(max_length=161)), (OK, {}, dict(total_tokens=0, max_tokens=0)),
                                               (UNSUPPORTED, dict(pages=1 << 26), {})])
def test_views_and_batches(status, view, batch):
    assert scored(view_of(**view), batch_of(**batch)) == status
    v, b = view_of(), batch_of()
    assert lib.b200kv_paged_attn_scored(C.byref(v), C.byref(b), None, 16, 0, None, 1 << 20, 0, None, 8, 0.1, 0, 0, 1 << 24, 1 << 40, None) == INVALID


def test_workspace():
    v = view_of()
    for tokens in (1, 7):
        b = batch_of(max_tokens=tokens)
        assert room(v, b, ranges=None) == size(v, b) and room(v, b, ranges=None, window=30, sinks=4) == size(v, b, window=30, sinks=4)
    b = batch_of(sequences=700, total_tokens=7000, max_tokens=40)
    rows = 7000 * 4 // 128 + 701                  # most row tiles there can be: their walks, twice, and bounds of every sequence
    assert 8 * (2 * rows + 700) <= room(v, b) - size(v, b) <= 8 * (2 * rows + 700) + 3 * 1024
    few = batch_of(max_tokens=1)
    assert room(v, few) == size(v, few)          # no chunks: nothing is laid out
    assert lib.b200kv_paged_attn_scored_workspace_bytes(C.byref(v), C.byref(b), None, 8, 0, 0) == 0


def test_tensors_that_are_refused():
    f, i = torch.zeros(4), torch.zeros(5, 2, dtype=torch.int32)
    for bad in (dict(slopes=f), dict(ranges=i), dict(slopes=f.half()), dict(ranges=i.long())):     # (no CUDA tensors)
        with pytest.raises(ValueError):
            paged.PagedScoring(**bad)
    assert paged.PagedScoring(cap=20.0).cap == 20.0

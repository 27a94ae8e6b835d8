"""Paged calls one behind the other under launch overlap, replayed from a graph, and again: the bits of the calls by themselves; bounds at zero."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import kv, paged
from test_paged_gpu import status  # noqa: F401

pytestmark = pytest.mark.gpu

MODES = [(128, 3, 32, 8, 2), (256, 1, 256, 12, 2), (128, 2, 32, 4, 2), (256, 0, 256, 6, 1)]      # d, mode, qblock, query heads, kv heads


class Layer:
    """A step of a layer: store, attention, weights, load, eviction in place."""

    def __init__(self, rng, d, mode, qblock, hq, heads, tokens, keep=90):
        self.pool = po.Pool(rng, [400, 131, 90, 700], d=d, heads=heads, page=16, mode=mode, qblock=qblock)
        self.view = self.pool.upload()
        self.first = [None if p is None else p.clone() for p in self.pool.dev]
        self.batch, self.starts = po.batch_of(self.pool, tokens)
        n, self.hq, self.keep = sum(tokens), hq, keep
        self.scale = d ** -0.5
        self.k, self.v = (to_dev(rng.standard_normal((n, heads * d)).astype(np.float16)) for _ in range(2))
        self.q = to_dev((1.5 * rng.standard_normal((n, hq, d))).astype(np.float16))
        self.ws = paged.paged_workspace(self.view, self.batch, hq, window=200, sinks=4)
        half = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
        self.results = {"out": half(n, hq, d), "lse": torch.zeros(n, hq, device="cuda"), "w": torch.zeros(4, heads, 700, device="cuda"), "key": half(n, heads, d), "value": half(n, heads, d),
                        "kept": torch.zeros(4, heads, keep, dtype=torch.int32, device="cuda"), "new_w": torch.zeros(4, heads, keep, device="cuda"),
                        "new_len": torch.zeros(4, dtype=torch.int32, device="cuda")}

    def reset(self):
        for p, b in zip(self.pool.dev, self.first):
            if p is not None:
                p.copy_(b)
        for t in self.results.values():
            t.zero_()

    def step(self, stream=None):
        r, a = self.results, dict(query_heads=self.hq, scale=self.scale, window=200, sinks=4, stream=stream)
        paged.launch_paged_store(self.view, self.batch, self.k, self.v, None, rope_mode=kv.RopeMode.NEOX_FULL, stream=stream)
        paged.launch_paged_attention(self.view, self.batch, self.q, r["out"], lse=r["lse"], workspace=self.ws, **a)
        paged.launch_paged_weights(self.view, self.batch, self.q, r["lse"], r["w"], **a)
        paged.launch_paged_load(self.view, self.batch, r["key"], r["value"], stream=stream)
        paged.launch_paged_evict(self.view, self.batch, self.pool.table_dev, r["w"], keep=self.keep, sinks=4, recent=30, kept=r["kept"], new_lengths=r["new_len"], new_weights=r["new_w"],
                                 stream=stream)

    def found(self):
        return [t.clone() for t in self.results.values()] + [p.clone() for p in self.pool.dev if p is not None]


@pytest.mark.parametrize("tokens", [[1, 1, 1, 1], [70, 1, 33, 2]])
@pytest.mark.parametrize("d,mode,qblock,hq,heads", MODES)
def test_a_step_under_launch_overlap(cuda, status, d, mode, qblock, hq, heads, tokens):
    layer = Layer(np.random.default_rng(d + mode), d, mode, qblock, hq, heads, tokens)
    layer.reset()
    torch.cuda.synchronize()
    layer.step()
    torch.cuda.synchronize()
    alone = layer.found()
    assert any(bool(t.any()) for t in alone[:1]) and bool((alone[5][0] >= 0).all())
    stream = torch.cuda.Stream()
    kv.set_launch_overlap(1)
    try:
        for _ in range(3):
            with torch.cuda.stream(stream):
                layer.reset()
                layer.step(stream)
            stream.synchronize()
            assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(alone, layer.found()))
    finally:
        kv.set_launch_overlap(0)
    assert int(status) == 0


@pytest.mark.parametrize("overlap", [0, 1])
@pytest.mark.parametrize("tokens", [[1, 1, 1, 1], [70, 1, 33, 2]])
def test_a_step_with_its_eviction_replayed_from_a_graph(cuda, status, tokens, overlap):
    layer = Layer(np.random.default_rng(5), 128, 3, 32, 8, 2, tokens)
    layer.reset()
    layer.step()
    torch.cuda.synchronize()
    alone = layer.found()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    kv.set_launch_overlap(overlap)
    try:
        with torch.cuda.graph(graph, stream=stream):
            layer.step()
    finally:
        kv.set_launch_overlap(0)
    for _ in range(3):
        layer.reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in zip(alone, layer.found()))
    assert int(status) == 0


@pytest.mark.parametrize("hq,tokens", [(2, [1, 1]), (8, [1, 4]), (8, [20, 3]), (12, [9, 40])])
@pytest.mark.parametrize("d,mode", [(128, 3), (256, 0)])
def test_a_batch_whose_lengths_are_bounded_by_zero(cuda, status, hq, tokens, d, mode):
    """Tokens of sequences that hold nothing see nothing, whatever kernel their number chooses."""
    pool = po.Pool(np.random.default_rng(1), [0, 0], d=d, heads=2, page=16, mode=mode, qblock=d, capacity=16)
    view = pool.upload()
    batch, _ = po.batch_of(pool, tokens, max_length=0, total_length=0)
    n = sum(tokens)
    q, out, lse, w = torch.randn(n, hq, d, device="cuda"), torch.full((n, hq, d), 3.0, device="cuda"), torch.zeros(n, hq, device="cuda"), torch.full((2, 2, 5), 3.0, device="cuda")
    paged.launch_paged_attention(view, batch, q, out, query_heads=hq, scale=0.1, lse=lse, workspace=paged.paged_workspace(view, batch, hq))
    paged.launch_paged_weights(view, batch, q, lse, w, query_heads=hq, scale=0.1)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all()) and bool((w == 3.0).all()) and int(status) == 0


def test_the_cut_of_a_large_batch_is_the_same_each_time(cuda, status):
    """More work than 2^24 of the 128ths in which it is counted: a sum in floating point, in the order in which threads come, would not be one number."""
    rng = np.random.default_rng(3)
    lengths, tokens = [15001, 9999, 15777, 12345, 3000, 1], [1531, 2047, 1999, 1777, 333, 1]
    pool = po.Pool(rng, lengths, d=128, heads=8, page=128, mode=0, qblock=128)
    view = pool.upload()
    batch, _ = po.batch_of(pool, tokens)
    q = torch.randn(sum(tokens), 32, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).half()
    ws, first = paged.paged_workspace(view, batch, 32), None
    for _ in range(12):
        out = torch.zeros(sum(tokens), 32, 128, device="cuda")
        paged.launch_paged_attention(view, batch, q, out, query_heads=32, scale=0.09, workspace=ws)
        first = out if first is None else first
        assert torch.equal(out, first)
    assert int(status) == 0

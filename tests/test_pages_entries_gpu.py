"""How many entries a call on a book may have: a captured one of a fixed size is filled up with entries that are left out."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from miinfer_b200 import paged
from test_pages_gpu import Both, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("slots", [3, 40, 1500])
def test_a_call_of_as_many_entries_as_slots(cuda, status, slots):
    """Forks and growth of a few sequences among entries that are left out, captured once and replayed over others."""
    b = Both(2 * slots + 20, 16, slots, 4, layers=1, mode=0, heads=1, qblock=128, seed=slots)
    b.fill([37])
    parents, children, grown, add = (torch.full((slots,), -1, dtype=torch.int32, device="cuda") for _ in range(4))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.launch_pages_fork(b.book, b.views, parents, children, workspace=b.workspace)
        paged.launch_pages_grow(b.book, grown, add, workspace=b.workspace)
    rng = np.random.default_rng(slots)
    for turn in range(4):
        of = [np.full(slots, -1, np.int32) for _ in range(4)]
        empty, full = np.flatnonzero(b.host.lengths == 0), np.flatnonzero(b.host.lengths)
        n = min(len(empty), 1 + 2 * turn)
        at = rng.choice(slots, n, replace=False)
        of[0][at], of[1][at] = rng.choice(full, n), empty[:n]
        at = rng.choice(slots, min(len(full), 2), replace=False)
        of[2][at], of[3][at] = full[:len(at)], rng.integers(0, 5, len(at))
        for t, a in zip((parents, children, grown, add), of):
            t.copy_(torch.from_numpy(a))
        graph.replay()
        b.host.fork(of[0].tolist(), of[1].tolist(), None, b.copy)
        b.host.grow(of[2].tolist(), of[3].tolist())
        b.check(status)


def test_more_entries_than_that(cuda, status):
    """Growth takes up to 8192 entries whatever the book's size, a fork as many as there are slots; both refuse more, and change nothing."""
    b = Both(20, 16, 3, 4, layers=1, mode=0, heads=1, qblock=128)
    b.fill([37])
    entries = [-1] * 8191 + [0]
    b.grow(entries, [5] * 8192)
    b.check(status)
    for call in (lambda: paged.launch_pages_grow(b.book, po.ints(entries + [0]), po.ints([1] * 8193), workspace=b.workspace),
                 lambda: paged.launch_pages_fork(b.book, b.views, po.ints([0] * 4), po.ints([-1, -1, -1, 1]), workspace=b.workspace)):
        with pytest.raises(paged._lib.B200KvError):
            call()
    b.check(status)
    b.fork([0, 0, 0], [-1, -1, 1])
    b.check(status)

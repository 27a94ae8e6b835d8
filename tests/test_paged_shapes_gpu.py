"""Accounts, tables and results of a paged call go by the shapes that its documentation names: one that is laid out for other heads or another count is refused,
not read with a stride that its number of elements suggests."""
import numpy as np
import pytest
import torch

import paged_oracle as po
from gpu_util import to_dev
from miinfer_b200 import paged
from test_paged_gpu import status  # noqa: F401

pytestmark = pytest.mark.gpu

f32 = lambda *s: torch.zeros(*s, device="cuda")
i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")


def made(rng):
    pool = po.Pool(rng, [40, 30, 25], d=128, heads=2, page=16, mode=3, qblock=32, spare=6)
    return pool, pool.upload()


@pytest.mark.parametrize("slots", [3, 5, 6, 9])
def test_an_account_of_more_slots_than_the_batch_has_sequences(cuda, status, slots):
    """A server's account of all its slots beside a batch of three of them: the first three rows count, with the stride they have."""
    rng = np.random.default_rng(slots)
    pool, view = made(rng)
    batch, starts = po.batch_of(pool, [3, 1, 2])
    q = rng.standard_normal((6, 8, 128)).astype(np.float16)
    _, lse, _ = po.attention(pool, q, starts, 0.1)
    before = rng.random((slots, 2, 50)).astype(np.float32)
    w = to_dev(before)
    paged.launch_paged_weights(view, batch, to_dev(q), to_dev(lse.astype(np.float32)), w, query_heads=8, scale=0.1)
    added, limit = po.weights(pool, q, lse.astype(np.float32), starts, 0.1)
    got = w.cpu().numpy()
    for s, length in enumerate(pool.lengths):
        assert (np.abs(got[s, :, :length] - before[s, :, :length] - added[s]) <= limit[s] + 2.0 ** -23 * got[s, :, :length]).all()
        assert np.array_equal(got[s, :, length:], before[s, :, length:])
    assert np.array_equal(got[3:], before[3:])
    # and the eviction reads it the same way, into tables and results of as many slots
    keep = 20
    target = i32(slots, 2)
    target[:3] = torch.from_numpy(pool.spare.reshape(3, 2).astype(np.int32)).cuda()
    kept, new_w = i32(slots, 2, keep).fill_(99), f32(slots, 2, keep).fill_(99)
    new_len = i32(slots).fill_(99)
    paged.launch_paged_evict(view, batch, target, w, keep=keep, sinks=1, recent=3, kept=kept, new_lengths=new_len, new_weights=new_w)
    for s, length in enumerate(pool.lengths):
        for h in range(2):
            want = po.evict(got[s, h], length, keep, 1, 3)
            assert np.array_equal(kept[s, h].cpu().numpy(), want)
            assert np.array_equal(new_w[s, h].cpu().numpy(), got[s, h, want])
    assert new_len.tolist() == [20, 20, 20] + [99] * (slots - 3) and bool((kept[3:] == 99).all()) and bool((new_w[3:] == 99).all())
    assert int(status) == 0


def test_shapes_that_are_refused(cuda):
    rng = np.random.default_rng(1)
    pool, view = made(rng)
    batch, _ = po.batch_of(pool, [3, 1, 2])
    q, lse = torch.zeros(6, 8, 128, dtype=torch.float16, device="cuda"), f32(6, 8)
    weigh = lambda w: paged.launch_paged_weights(view, batch, q, lse, w, query_heads=8, scale=0.1)
    for w in (f32(3, 1, 80), f32(3, 3, 40), f32(3, 80), f32(240), f32(2, 2, 60), f32(3, 2, 39), f32(1, 3, 2, 40), f32(6, 1, 40), f32(2, 3, 40)):
        with pytest.raises(ValueError):
            weigh(w)
    evict = lambda table=i32(3, 2), w=f32(3, 2, 40), kept=i32(3, 2, 20), new_weights=f32(3, 2, 20), lengths=i32(3): paged.launch_paged_evict(
        view, batch, table, w, keep=20, kept=kept, new_lengths=lengths, new_weights=new_weights)
    for call in (lambda: evict(table=i32(6)), lambda: evict(table=i32(2, 3)), lambda: evict(table=i32(1, 3, 2)), lambda: evict(w=f32(2, 3, 40)), lambda: evict(w=f32(3, 80)),
                 lambda: evict(kept=i32(3, 2, 21)), lambda: evict(kept=i32(3, 1, 40)), lambda: evict(kept=i32(120)), lambda: evict(kept=i32(2, 2, 30)),
                 lambda: evict(new_weights=f32(3, 2, 32)), lambda: evict(new_weights=f32(3, 4, 20)), lambda: evict(new_weights=f32(120)), lambda: evict(lengths=i32(2))):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("call", ["weights", "evict"])
def test_a_view_without_heads_is_an_error(cuda, call):
    pool, _ = made(np.random.default_rng(2))
    view, (batch, _) = paged.PagedView(), po.batch_of(pool, [3, 1, 2])
    with pytest.raises((ValueError, RuntimeError)):
        if call == "weights":
            paged.launch_paged_weights(view, batch, torch.zeros(6, 8, 128, dtype=torch.float16, device="cuda"), f32(6, 8), f32(3, 2, 40), query_heads=8, scale=0.1)
        else:
            paged.launch_paged_evict(view, batch, i32(3, 2), f32(3, 2, 40), keep=20, kept=i32(3, 2, 20), new_lengths=i32(3))

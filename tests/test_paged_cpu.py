"""What the entry points over a paged cache refuse, and the size of the attention's workspace; no GPU needed: every refused call ends at its arguments."""
import ctypes as C
import random

import pytest
import torch

from miinfer_b200 import kv, paged
from miinfer_b200._lib import PagedBatch, PagedView, lib, native

OK, INVALID, UNSUPPORTED, DEVICE, WORKSPACE, RANGE = 0, -1, -2, -4, -5, -6
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the call would be launched over addresses that are none")


def view_of(**k):
    return PagedView(**{**dict(key_q8=4096, key_scales=8192, value_q8=16384, value_scales=32768, pages=40, page_size=16, kv_heads=2, head_dim=128, qblock=32, quant_mode=3), **k})


def batch_of(**k):
    return PagedBatch(**{**dict(page_table=4096, query_starts=8192, lengths=12288, sequences=3, max_pages=10, total_tokens=9, max_tokens=7, max_length=160, total_length=200), **k})


def store(v, b, key=4096, value=8192, dtype=0, weight=None, rope=1, theta=1e6, epsilon=1e-6, positions=None):
    return lib.b200kv_paged_store(C.byref(v), C.byref(b), key, value, dtype, weight, rope, theta, epsilon, positions, None)


def load(v, b, key=4096, value=8192):
    return lib.b200kv_paged_load(C.byref(v), C.byref(b), key, value, None)


def attend(v, b, q=4096, q_dtype=0, gate=None, out=8192, out_dtype=0, lse=None, query_heads=8, scale=0.1, window=0, sinks=0, workspace=1 << 20, room=1 << 40):
    return lib.b200kv_paged_attn(C.byref(v), C.byref(b), q, q_dtype, gate, out, out_dtype, lse, query_heads, scale, window, sinks, workspace, room, None)


def weigh(v, b, q=4096, q_dtype=0, lse=8192, weights=16384, stride=160, query_heads=8, scale=0.1, window=0, sinks=0, observe=0):
    return lib.b200kv_paged_weights(C.byref(v), C.byref(b), q, q_dtype, lse, weights, stride, query_heads, scale, window, sinks, observe, None)


def evict(v, b, target=1 << 14, pages=4, weights=1 << 20, stride=160, keep=64, sinks=4, recent=16, kept=1 << 16, new_weights=1 << 24, new_lengths=1 << 18):
    return lib.b200kv_paged_evict(C.byref(v), C.byref(b), target, pages, weights, stride, keep, sinks, recent, kept, new_weights, new_lengths, None)


CALLS = [store, load, attend, weigh, evict]


def size(v, b, heads=8, window=0, sinks=0):
    return lib.b200kv_paged_attn_workspace_bytes(C.byref(v), C.byref(b), heads, window, sinks)


@no_gpu
@pytest.mark.parametrize("call", CALLS)
def test_a_call_that_is_right_ends_at_the_missing_device(call):
    assert call(view_of(), batch_of()) == DEVICE


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("status,change", [
    (INVALID, dict(pages=0)), (INVALID, dict(kv_heads=0)), (INVALID, dict(quant_mode=4)),
    (UNSUPPORTED, dict(page_size=8)), (UNSUPPORTED, dict(page_size=48)), (UNSUPPORTED, dict(page_size=512)), (UNSUPPORTED, dict(page_size=0)),
    (UNSUPPORTED, dict(head_dim=64)), (UNSUPPORTED, dict(head_dim=96)), (UNSUPPORTED, dict(qblock=64)), (UNSUPPORTED, dict(qblock=0)),
    (UNSUPPORTED, dict(pages=1 << 31)), (UNSUPPORTED, dict(kv_heads=1 << 16)),
    (INVALID, dict(key_q8=None)), (INVALID, dict(key_scales=None)), (INVALID, dict(value_q8=None)), (INVALID, dict(value_scales=None)),
    (INVALID, dict(key_q8=4104)), (INVALID, dict(value_scales=32770)),
    (INVALID, dict(quant_mode=0)), (INVALID, dict(quant_mode=1)), (INVALID, dict(quant_mode=2)), (INVALID, dict(quant_mode=0, key_f16=64, value_f16=72)),
])
def test_views_that_no_call_takes(call, status, change):
    assert call(view_of(**change), batch_of()) == status


@pytest.mark.parametrize("call", [attend, weigh])
def test_pools_of_more_rows_than_a_coordinate_counts(call):
    assert call(view_of(pages=1 << 26), batch_of()) == UNSUPPORTED


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("status,change", [
    (INVALID, dict(page_table=None)), (INVALID, dict(query_starts=None)), (INVALID, dict(lengths=None)), (INVALID, dict(page_table=4098)), (INVALID, dict(lengths=12289)),
    (INVALID, dict(max_pages=0)), (UNSUPPORTED, dict(sequences=8193)), (INVALID, dict(total_tokens=1 << 31)), (INVALID, dict(max_length=1 << 31, max_pages=1 << 31)),
    (INVALID, dict(max_tokens=10)), (RANGE, dict(max_length=161)),
])
def test_batches_that_no_call_takes(call, status, change):
    assert call(view_of(), batch_of(**change)) == status


@pytest.mark.parametrize("entry,more", [("store", 9), ("load", 3), ("attn", 13), ("weights", 11), ("evict", 11)])
def test_no_view_or_batch(entry, more):
    f = getattr(lib, "b200kv_paged_" + entry)
    rest = [t(0) if t is not C.c_void_p else None for t in f.argtypes[2:]]
    assert len(rest) == more
    assert f(None, C.byref(batch_of()), *rest) == INVALID and f(C.byref(view_of()), None, *rest) == INVALID


@pytest.mark.parametrize("status,call,change", [
    (INVALID, store, dict(key=None)), (INVALID, store, dict(value=None)), (INVALID, store, dict(dtype=2)), (INVALID, store, dict(dtype=-1)),
    (INVALID, store, dict(rope=3)), (INVALID, store, dict(rope=-1)), (INVALID, store, dict(theta=0.0)), (INVALID, store, dict(theta=-1.0)),
    (INVALID, store, dict(theta=float("nan"))), (INVALID, store, dict(epsilon=float("inf"))),
    (INVALID, load, dict(key=None, value=None)), (INVALID, load, dict(key=4104)), (INVALID, load, dict(value=8194)),
    (INVALID, attend, dict(q=None)), (INVALID, attend, dict(out=None)), (INVALID, attend, dict(q_dtype=2)), (INVALID, attend, dict(out_dtype=-1)),
    (INVALID, attend, dict(q=4104)), (INVALID, attend, dict(out=8200)), (INVALID, attend, dict(gate=8)), (INVALID, attend, dict(workspace=(1 << 20) + 8)), (INVALID, attend, dict(lse=2)),
    (INVALID, attend, dict(query_heads=0)), (INVALID, attend, dict(query_heads=7)), (UNSUPPORTED, attend, dict(query_heads=18)),
    (INVALID, attend, dict(scale=0.0)), (INVALID, attend, dict(scale=-0.1)), (INVALID, attend, dict(scale=float("nan"))), (INVALID, attend, dict(scale=float("inf"))),
    (WORKSPACE, attend, dict(workspace=None)), (WORKSPACE, attend, dict(room=0)), (WORKSPACE, attend, dict(room=size(view_of(), batch_of()) - 1)),
    (INVALID, weigh, dict(q=None)), (INVALID, weigh, dict(lse=None)), (INVALID, weigh, dict(weights=None)), (INVALID, weigh, dict(q_dtype=2)), (INVALID, weigh, dict(q=4104)),
    (INVALID, weigh, dict(lse=8194)), (INVALID, weigh, dict(weights=16386)), (INVALID, weigh, dict(stride=159)), (INVALID, weigh, dict(query_heads=0)),
    (INVALID, weigh, dict(query_heads=7)), (UNSUPPORTED, weigh, dict(query_heads=18)), (INVALID, weigh, dict(scale=0.0)), (INVALID, weigh, dict(scale=float("nan"))),
    (INVALID, evict, dict(target=None)), (INVALID, evict, dict(weights=None)), (INVALID, evict, dict(kept=None)), (INVALID, evict, dict(new_lengths=None)),
    (INVALID, evict, dict(target=(1 << 14) + 2)), (INVALID, evict, dict(new_weights=(1 << 24) + 2)), (INVALID, evict, dict(keep=0, sinks=0, recent=0)),
    (INVALID, evict, dict(sinks=49)), (INVALID, evict, dict(sinks=0xffffffff, recent=65)), (INVALID, evict, dict(stride=159)), (RANGE, evict, dict(pages=3)), (RANGE, evict, dict(keep=1 << 31)),
    (INVALID, evict, dict(new_lengths=12288)),                                   # the batch's own lengths
    (INVALID, evict, dict(target=4096, pages=9)),                                # in place, with rows of another width
    (INVALID, evict, dict(new_weights=(1 << 20) + 4 * (3 * 2 * 160 - 1))),       # overlaps the last weight
    (INVALID, evict, dict(new_weights=(1 << 20) - 4 * (3 * 2 * 64 - 1))),        # its last one overlaps the first
])
def test_arguments_that_a_call_refuses(status, call, change):
    assert call(view_of(), batch_of(), **change) == status


@no_gpu
@pytest.mark.parametrize("call,change", [(evict, dict(new_weights=(1 << 20) + 4 * 3 * 2 * 160)), (evict, dict(new_weights=(1 << 20) - 4 * 3 * 2 * 64)), (evict, dict(new_weights=None)),
                                         (evict, dict(sinks=48)), (evict, dict(target=4096, pages=10)), (evict, dict(keep=1 << 20, pages=10)), (store, dict(theta=-1.0, rope=0)), (load, dict(value=None)),
                                         (attend, dict(room=size(view_of(), batch_of()))), (attend, dict(query_heads=16)), (weigh, dict(window=5, sinks=3, observe=1))])
def test_arguments_at_the_edge_of_what_a_call_takes(call, change):
    assert call(view_of(), batch_of(), **change) == DEVICE


@pytest.mark.parametrize("call", CALLS)
def test_a_batch_without_work_is_no_launch(call):
    assert call(view_of(), batch_of(sequences=0, page_table=None, query_starts=None, lengths=None, total_tokens=0, max_tokens=0, max_length=0, max_pages=0)) == OK
    if call is not evict:
        assert call(view_of(), batch_of(total_tokens=0, max_tokens=0)) == OK
    if call in (attend, weigh):
        assert call(view_of(), batch_of(max_tokens=0)) == OK
        assert call(view_of(), batch_of(max_tokens=0, max_length=0), **(dict(workspace=None, room=0) if call is attend else {})) == OK


def test_the_workspace_of_nothing_and_of_what_is_refused():
    assert lib.b200kv_paged_attn_workspace_bytes(None, C.byref(batch_of()), 8, 0, 0) == 0
    assert lib.b200kv_paged_attn_workspace_bytes(C.byref(view_of()), None, 8, 0, 0) == 0
    assert size(view_of(), batch_of(), heads=0) == 0 and size(view_of(), batch_of(), heads=7) == 0 and size(view_of(kv_heads=0), batch_of()) == 0
    assert size(view_of(), batch_of(sequences=0, total_tokens=0, max_tokens=0, max_length=0, total_length=0)) > 0
    assert paged.paged_workspace(view_of(), batch_of(), 8, device="cpu").numel() == size(view_of(), batch_of())


def test_a_workspace_does_for_every_batch_within_the_bounds():
    rng = random.Random(4)
    lower = lambda n: rng.choice([n, max(n - 1, 0), rng.randint(0, n), min(n, 1)])
    for _ in range(3000):
        d, heads, group = rng.choice([128, 256]), rng.choice([1, 2, 8]), rng.randint(1, 8)
        v = view_of(head_dim=d, qblock=d, kv_heads=heads)
        sequences, length = rng.choice([1, 2, 5, 64, 300]), rng.choice([1, 100, 128, 129, 5000, 200000])
        tokens = rng.choice([1, 2, 8, 9, 100, 4000])
        total = rng.randint(tokens, sequences * tokens)
        sums = rng.choice([0, sequences * length, rng.randint(length, sequences * length)])
        window, sinks = rng.choice([0, 0, 1, 100, 4096]), rng.choice([0, 4, 200])
        bounds = dict(sequences=sequences, total_tokens=total, max_tokens=tokens, max_length=length, total_length=sums, max_pages=1 << 20)
        small = {k: lower(n) for k, n in bounds.items() if k not in ("max_pages", "total_length")}
        small["max_tokens"] = min(small["max_tokens"], small["total_tokens"])
        small["total_length"] = rng.choice([0, small["sequences"] * small["max_length"]])
        if sums and (small["total_length"] or small["sequences"] * small["max_length"]) > sums:
            small["total_length"] = sums
        assert size(v, batch_of(**{**bounds, **small}), heads * group, window, sinks) <= size(v, batch_of(**bounds), heads * group, window, sinks), (bounds, small, heads, group, window, sinks)


# ---- through Python ---------------------------------------------------------------------------------------------------------------------


def test_python_views_and_batches_are_checked():
    plane, q8, scales = torch.zeros(4, 2, 16, 128, dtype=torch.float16), torch.zeros(4, 2, 16, 128, dtype=torch.int8), torch.zeros(4, 2, 16, 4, dtype=torch.float16)
    f, q = kv.KvCacheQuantMode.kFp16Fp16, kv.KvCacheQuantMode.kQ8Q8
    for args in [(plane, None, plane, None, f), (plane, None, plane, None, q), (q8, None, q8, None, q), (q8, scales, q8, scales[:3], q), (q8, scales, q8, scales.float(), q),
                 (q8, scales, q8, torch.zeros(4, 2, 16, 3, dtype=torch.float16), q), (plane, None, plane[:2], None, f), (plane[0], None, plane[0], None, f), (q8, scales, q8, scales, q)]:
        with pytest.raises(ValueError):        # (the right ones among them are not CUDA tensors)
            paged.PagedView.of(*args)
    table, starts, lengths = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    bounds = dict(total_tokens=1, max_tokens=1, max_length=1)
    for args in [(table, starts, lengths), (table[0], starts, lengths), (table, starts[:3], lengths), (table, starts, lengths[:2]), (table.long(), starts, lengths)]:
        with pytest.raises(ValueError):
            paged.PagedBatch(*args, **bounds)
    with pytest.raises(RuntimeError):
        paged.PagedKvCache(0, 16)
    with pytest.raises(ValueError):
        paged.PagedKvCache(4, 16, head_dim=128, qblock=48, device="cpu")
    cache = paged.PagedKvCache(4, 16, kv.KvCacheQuantMode.kQ8Fp16, kv_heads=2, head_dim=128, qblock=32, device="cpu")
    assert [tuple(t.shape) for t in cache.planes()] == [(4, 2, 16, 128), (4, 2, 16, 4), (4, 2, 16, 128)]
    assert [t.dtype for t in cache.planes()] == [torch.int8, torch.float16, torch.float16]


def test_python_calls_take_views_batches_and_cuda_tensors_only():
    t, v, b = torch.zeros(64), view_of(), batch_of()
    for not_it in (None, 7, b"x" * 256, v, torch.zeros(256, dtype=torch.uint8), C.byref(b)):
        with pytest.raises(TypeError):
            paged.launch_paged_load(v, not_it, t, t)
        with pytest.raises(TypeError):
            paged.launch_paged_load(b if not_it is v else not_it, b, t, t)
    for call in (lambda x: paged.launch_paged_store(v, b, x, x, None), lambda x: paged.launch_paged_load(v, b, x, None),
                 lambda x: paged.launch_paged_attention(v, b, x, x, query_heads=8, scale=0.1, workspace=x), lambda x: paged.launch_paged_weights(v, b, x, x, x, query_heads=8, scale=0.1),
                 lambda x: paged.launch_paged_evict(v, b, x, x, keep=4, kept=x, new_lengths=x)):
        with pytest.raises(ValueError, match="contiguous CUDA tensor"):
            call(t)
        with pytest.raises(TypeError):
            call("rows")
    with pytest.raises(ValueError):
        paged.launch_paged_store(v, b, None, None, None)
    with pytest.raises(TypeError):
        native.paged_load(v, b, t)

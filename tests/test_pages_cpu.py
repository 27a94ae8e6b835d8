"""What the calls on a book of pages refuse, and the size of their workspace; no GPU needed: every refused call ends at its arguments."""
import ctypes as C

import pytest
import torch

from miinfer_b200._lib import PageBook, PagedView, lib
from test_paged_cpu import DEVICE, INVALID, OK, UNSUPPORTED, WORKSPACE, no_gpu, view_of

BIG = 1 << 40


def book_of(**k):
    return PageBook(**{**dict(refs=1 << 20, tables=1 << 21, lengths=1 << 22, pages=40, page_size=16, slots=6, max_pages=10), **k})


def views_of(count=2, **k):
    return (PagedView * max(count, 1))(*[view_of(**k) for _ in range(count)])


def grow(b, slots=4096, add=8192, count=5, workspace=1 << 24, room=BIG):
    return lib.b200kv_pages_grow(C.byref(b), slots, add, count, workspace, room, None)


def fork(b, views=None, layers=2, parents=4096, children=8192, at=None, count=5, workspace=1 << 24, room=BIG):
    return lib.b200kv_pages_fork(C.byref(b), views_of() if views is None else views, layers, parents, children, at, count, workspace, room, None)


def free(b, slots=4096, count=5):
    return lib.b200kv_pages_free(C.byref(b), slots, count, None)


def compact(b, views=None, layers=2, moved=4096, workspace=1 << 24, room=BIG):
    return lib.b200kv_pages_compact(C.byref(b), views_of() if views is None else views, layers, moved, workspace, room, None)


def copy(source=None, target=None, layers=2, sources=4096, targets=8192, count=5):
    return lib.b200kv_pages_copy(views_of() if source is None else source, views_of() if target is None else target, layers, sources, targets, count, None)


CALLS = [grow, fork, free, compact]


@no_gpu
def test_calls_that_are_right_end_at_the_missing_device():
    assert [call(book_of()) for call in CALLS] == [DEVICE] * 4 and copy() == DEVICE
    assert copy(target=views_of(pages=7)) == DEVICE                      # pools of another size
    assert fork(book_of(), at=1 << 14) == DEVICE and fork(book_of(), views_of(128), 128) == DEVICE


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("status,change", [
    (INVALID, dict(pages=0)), (INVALID, dict(slots=0)), (INVALID, dict(max_pages=0)), (UNSUPPORTED, dict(page_size=8)), (UNSUPPORTED, dict(page_size=48)),
    (UNSUPPORTED, dict(page_size=512)), (UNSUPPORTED, dict(pages=1 << 31)), (UNSUPPORTED, dict(slots=8193)), (UNSUPPORTED, dict(max_pages=1 << 22)),
    (INVALID, dict(refs=None)), (INVALID, dict(tables=None)), (INVALID, dict(lengths=None)), (INVALID, dict(refs=(1 << 20) + 4)), (INVALID, dict(tables=(1 << 21) + 2)),
    (INVALID, dict(lengths=(1 << 22) + 1)),
])
def test_books_that_no_call_takes(call, status, change):
    assert call(book_of(**change)) == status


@pytest.mark.parametrize("status,call,change", [
    (INVALID, grow, dict(slots=None)), (INVALID, grow, dict(add=None)), (INVALID, grow, dict(slots=4098)), (INVALID, grow, dict(count=8193)), (INVALID, grow, dict(workspace=(1 << 24) + 8)),
    (WORKSPACE, grow, dict(workspace=None)), (WORKSPACE, grow, dict(room=0)), (OK, grow, dict(count=0, slots=None)),
    (INVALID, grow, dict(add=1 << 22)), (INVALID, grow, dict(add=(1 << 22) + 20)), (INVALID, grow, dict(slots=(1 << 20) - 16)), (INVALID, grow, dict(slots=(1 << 21) + 4 * 59)),
    (INVALID, fork, dict(parents=None)), (INVALID, fork, dict(children=None)), (INVALID, fork, dict(at=2)), (INVALID, fork, dict(count=7)), (INVALID, fork, dict(layers=0)),
    (INVALID, fork, dict(at=1 << 22)), (INVALID, fork, dict(children=1 << 22)), (INVALID, fork, dict(parents=(1 << 20) + 4 * 39)), (WORKSPACE, fork, dict(workspace=None)), (WORKSPACE, fork, dict(room=100)),
    (UNSUPPORTED, fork, dict(views=views_of(129), layers=129)), (INVALID, fork, dict(views=views_of(pages=41))), (INVALID, fork, dict(views=views_of(page_size=32))),
    (UNSUPPORTED, fork, dict(views=views_of(head_dim=64))), (INVALID, fork, dict(views=views_of(key_q8=None))), (OK, fork, dict(count=0)),
    (INVALID, free, dict(slots=None)), (INVALID, free, dict(slots=4097)), (INVALID, free, dict(slots=1 << 22)), (INVALID, free, dict(count=1 << 31)), (OK, free, dict(count=0)),
    (INVALID, compact, dict(moved=None)), (INVALID, compact, dict(moved=1 << 20)), (INVALID, compact, dict(moved=(1 << 20) - 4 * 39)), (INVALID, compact, dict(moved=1 << 21)),
    (INVALID, compact, dict(moved=(1 << 24) + 256)), (WORKSPACE, compact, dict(workspace=None)), (WORKSPACE, compact, dict(room=8)), (INVALID, compact, dict(layers=0)),
])
def test_arguments_that_a_call_refuses(status, call, change):
    assert call(book_of(), **change) == status


@pytest.mark.parametrize("status,change", [
    (INVALID, dict(sources=None)), (INVALID, dict(targets=None)), (INVALID, dict(targets=8194)), (INVALID, dict(layers=0)), (OK, dict(count=0)), (INVALID, dict(count=1 << 31)),
    (INVALID, dict(target=views_of(page_size=32))), (INVALID, dict(target=views_of(kv_heads=4))), (INVALID, dict(target=views_of(qblock=128))),
    (INVALID, dict(target=views_of(quant_mode=2, key_f16=4096))), (INVALID, dict(source=(PagedView * 2)(view_of(), view_of(kv_heads=4)))),
    (INVALID, dict(source=(PagedView * 2)(view_of(), view_of(pages=41)))), (UNSUPPORTED, dict(source=(PagedView * 2)(view_of(), view_of(page_size=24)))),
])
def test_copies_that_are_refused(status, change):
    assert copy(**change) == status


def test_no_book_and_no_views():
    assert lib.b200kv_pages_grow(None, 4096, 8192, 1, 1 << 24, BIG, None) == INVALID and lib.b200kv_pages_free(None, 4096, 1, None) == INVALID
    assert lib.b200kv_pages_fork(C.byref(book_of()), None, 2, 4096, 8192, None, 1, 1 << 24, BIG, None) == INVALID
    assert lib.b200kv_pages_compact(C.byref(book_of()), None, 2, 4096, 1 << 24, BIG, None) == INVALID
    assert lib.b200kv_pages_copy(None, views_of(), 2, 4096, 8192, 1, None) == INVALID and lib.b200kv_pages_copy(views_of(), None, 2, 4096, 8192, 1, None) == INVALID


def test_size_of_the_workspace():
    size = lambda **k: lib.b200kv_pages_workspace_bytes(C.byref(book_of(**k)))
    assert size(pages=0) == 0 and lib.b200kv_pages_workspace_bytes(None) == 0
    for pages, slots in ((1, 1), (40, 6), (4096, 8192), (4097, 1), (1 << 20, 77)):
        n = size(pages=pages, slots=slots)
        assert n % 256 == 0 and 4 * (3 * pages + slots + -(-pages // 4096)) + 256 <= n < 4 * (3 * pages + slots + -(-pages // 4096)) + 7 * 256
        assert grow(book_of(pages=pages, slots=slots), slots=16, add=32, count=1, room=n - 1) == WORKSPACE
    assert torch.cuda.is_available() or grow(book_of(), room=size()) == DEVICE

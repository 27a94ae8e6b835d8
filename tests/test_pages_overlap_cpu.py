"""A workspace that lies over what its call reads or changes is refused before a device is looked for; no GPU needed."""
import ctypes as C

import pytest

from miinfer_b200._lib import lib
from test_paged_cpu import DEVICE, INVALID, no_gpu
from test_pages_cpu import book_of, compact, fork, grow

ROOM = lib.b200kv_pages_workspace_bytes(C.byref(book_of()))
# the book's arrays: refs 40 words at 1 << 20, tables 60 words at 1 << 21, lengths 6 words at 1 << 22
OVER_BOOK = [(1 << 20) - ROOM + 16, 1 << 20, (1 << 20) + 4 * 36, (1 << 21) - ROOM + 16, (1 << 21) + 4 * 56, (1 << 22) - ROOM + 16, (1 << 22) + 16]
BESIDE = [(1 << 20) - ROOM, (1 << 20) + 4 * 40, (1 << 21) - ROOM, (1 << 21) + 4 * 60, (1 << 22) - ROOM, (1 << 22) + 32]


@pytest.mark.parametrize("call", [grow, fork, compact])
def test_workspace_over_the_book(call):
    assert [call(book_of(), workspace=at) for at in OVER_BOOK] == [INVALID] * len(OVER_BOOK)


@pytest.mark.parametrize("call,names", [(grow, ["slots", "add"]), (fork, ["parents", "children", "at"])])
def test_workspace_over_the_entries(call, names):
    for name in names:
        assert call(book_of(), **{name: 1 << 24}) == INVALID
        assert call(book_of(), **{name: (1 << 24) + ROOM - 4}) == INVALID
        assert call(book_of(), **{name: (1 << 24) - 4}) == INVALID


@no_gpu
def test_workspace_beside_them():
    for call in (grow, fork, compact):
        assert [call(book_of(), workspace=at) for at in BESIDE] == [DEVICE] * len(BESIDE)
    for call, names in ((grow, ["slots", "add"]), (fork, ["parents", "children", "at"])):
        for name in names:
            assert call(book_of(), **{name: (1 << 24) + ROOM}) == DEVICE and call(book_of(), **{name: (1 << 24) - 4 * 5}) == DEVICE

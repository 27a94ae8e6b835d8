"""A paged KV cache: many sequences in one pool of pages, served in ragged batches (b200kv_paged_*; no counterpart in the
reference, which keeps one session resident).

A pool's planes are [page][kv_head][slot][...]; position j of a sequence lies in slot j % page_size of page
page_table[sequence][j // page_size].  A batch names the sequences' pages, the rows of the activations that are their newest
tokens, and their lengths, all in device memory, so that a captured graph replays with whatever these then hold; the host-side
bounds beside them size the launches.  A layer of a serving step is `launch_paged_store` and `launch_paged_attention`; where a
cache is to stay bounded, `launch_paged_weights` keeps account of what the tokens looked at and `launch_paged_evict` brings a
sequence back to the positions that were looked at most.  Tensors are contiguous CUDA tensors of the current device.
Argument errors raise B200KvError or ValueError.
"""
from __future__ import annotations

import ctypes as C
import enum
from typing import Optional, Sequence

import torch

from . import _lib
from ._lib import check, lib, native
from .kv import KvCacheQuantMode, RopeMode

__all__ = ["PagedView", "PagedBatch", "PagedKvCache", "PagedScoring", "paged_workspace", "launch_paged_store", "launch_paged_load", "launch_paged_attention",
           "launch_paged_weights", "launch_paged_evict", "RotaryLayout", "RotaryScaling", "RotaryTable", "launch_paged_rotary", "PageBook", "pages_workspace",
           "launch_pages_grow", "launch_pages_fork", "launch_pages_free", "launch_pages_compact", "launch_pages_copy", "STATUS_BAD_PAGE", "STATUS_BAD_BOUND",
           "STATUS_BAD_SLOT", "STATUS_NO_PAGE"]

STATUS_BAD_PAGE, STATUS_BAD_BOUND, STATUS_BAD_SLOT, STATUS_NO_PAGE = 16, 32, 64, 128      # bits of the word registered with kv.set_status_word


class PagedView(_lib.PagedView):
    """b200kv_paged_view; `of` builds one from the planes' tensors and keeps them."""

    @staticmethod
    def of(key: torch.Tensor, key_scales: Optional[torch.Tensor], value: torch.Tensor, value_scales: Optional[torch.Tensor],
           quant_mode: KvCacheQuantMode) -> "PagedView":
        """key/value: [pages][kv_heads][page_size][head_dim] of int8 or fp16, scales (int8 sides): [...][head_dim / qblock] of fp16."""
        mode = KvCacheQuantMode(quant_mode)
        q8 = (mode in (KvCacheQuantMode.kQ8Fp16, KvCacheQuantMode.kQ8Q8), mode in (KvCacheQuantMode.kFp16Q8, KvCacheQuantMode.kQ8Q8))
        blocks = set()
        for plane, scales, is_q8 in ((key, key_scales, q8[0]), (value, value_scales, q8[1])):
            if plane.dim() != 4 or plane.shape != key.shape or plane.dtype != (torch.int8 if is_q8 else torch.float16):
                raise ValueError("planes are [pages][kv_heads][page_size][head_dim] of the mode's types")
            tensors = [plane]
            if is_q8:
                if (scales is None or scales.dtype != torch.float16 or scales.dim() != 4 or scales.shape[:3] != plane.shape[:3] or scales.shape[3] == 0
                        or plane.shape[3] % scales.shape[3]):
                    raise ValueError("scales are fp16 [pages][kv_heads][page_size][head_dim / qblock]")
                blocks.add(plane.shape[3] // scales.shape[3])
                tensors.append(scales)
            if not all(t.is_cuda and t.is_contiguous() and t.device == key.device for t in tensors):
                raise ValueError("expected contiguous CUDA tensors of one device")
        if len(blocks) > 1:
            raise ValueError("both sides have the same qblock")
        pages, heads, page_size, dim = key.shape
        ptr = lambda t, want: t.data_ptr() if want else None
        view = PagedView(ptr(key, not q8[0]), ptr(value, not q8[1]), ptr(key, q8[0]), ptr(key_scales, q8[0]), ptr(value, q8[1]), ptr(value_scales, q8[1]),
                         pages, page_size, heads, dim, blocks.pop() if blocks else dim, int(mode))
        view.planes, view.device_index = (key, key_scales, value, value_scales), key.device.index
        return view


class PagedBatch(_lib.PagedBatch):
    """b200kv_paged_batch over int32 CUDA tensors: page_table [sequences][max_pages], query_starts [sequences + 1], lengths [sequences].

    total_tokens: rows of the activations; max_tokens, max_length, total_length: upper bounds of a sequence's new tokens, of a
    length and of the sum of the lengths (0: sequences * max_length).  Lengths count the new tokens."""

    def __init__(self, page_table: torch.Tensor, query_starts: torch.Tensor, lengths: torch.Tensor, *, total_tokens: int, max_tokens: int,
                 max_length: int, total_length: int = 0):
        sequences = lengths.numel()
        if page_table.dim() != 2 or page_table.shape[0] != sequences or query_starts.numel() != sequences + 1:
            raise ValueError("page_table [sequences][pages], query_starts [sequences + 1], lengths [sequences]")
        for t in (page_table, query_starts, lengths):
            if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.device != page_table.device:
                raise ValueError("expected contiguous int32 CUDA tensors of one device")
        for name, n in (("total_tokens", total_tokens), ("max_tokens", max_tokens), ("max_length", max_length), ("total_length", total_length)):
            if not 0 <= int(n) < (1 << 31 if name != "total_length" else 1 << 63):
                raise ValueError(f"{name} out of range")
        super().__init__(page_table.data_ptr(), query_starts.data_ptr(), lengths.data_ptr(), sequences, page_table.shape[1], int(total_tokens),
                         int(max_tokens), int(max_length), int(total_length))
        self.tensors, self.device_index = (page_table, query_starts, lengths), page_table.device.index


class PagedKvCache:
    """Owns one layer's pool: `pages` pages of `page_size` positions (16, 32, 64, 128 or 256).  Which sequence has which page is the caller's."""

    def __init__(self, pages: int, page_size: int, quant_mode: KvCacheQuantMode = KvCacheQuantMode.kFp16Fp16, *, kv_heads: int = 4, head_dim: int = 256,
                 qblock: Optional[int] = None, device: Optional[torch.device] = None):
        if pages <= 0:
            raise RuntimeError("PagedKvCache: pages must be > 0")
        self.pages, self.page_size, self.kv_heads, self.head_dim = int(pages), int(page_size), int(kv_heads), int(head_dim)
        self.qblock = int(qblock if qblock is not None else head_dim)
        self.quant_mode = KvCacheQuantMode(quant_mode)
        if self.head_dim % self.qblock:
            raise ValueError("qblock must divide head_dim")
        dev = device or torch.device("cuda", torch.cuda.current_device())
        shape, blocks = (self.pages, self.kv_heads, self.page_size, self.head_dim), self.head_dim // self.qblock
        side = lambda q8: (torch.zeros(shape, dtype=torch.int8 if q8 else torch.float16, device=dev),
                           torch.zeros(*shape[:3], blocks, dtype=torch.float16, device=dev) if q8 else None)
        self.key, self.key_scales = side(self.quant_mode in (KvCacheQuantMode.kQ8Fp16, KvCacheQuantMode.kQ8Q8))
        self.value, self.value_scales = side(self.quant_mode in (KvCacheQuantMode.kFp16Q8, KvCacheQuantMode.kQ8Q8))

    def planes(self):
        return [t for t in (self.key, self.key_scales, self.value, self.value_scales) if t is not None]

    def view(self) -> PagedView:
        return PagedView.of(self.key, self.key_scales, self.value, self.value_scales, self.quant_mode)


class PagedScoring(_lib.PagedScoring):
    """b200kv_paged_scoring: scores cap * tanh(x / cap) in place of x = scale * q.k (cap 0: x), less slopes[head] * |i - j| (fp32 [query_heads]), and ranges (int32
    [total_tokens][2]): token t sees positions ranges[t][0] <= j < ranges[t][1] in place of j <= its own, as documents that do not see one another ask for, or a prefix that
    sees itself in both directions."""

    def __init__(self, *, cap: float = 0.0, slopes: Optional[torch.Tensor] = None, ranges: Optional[torch.Tensor] = None):
        for name, t, dtype, dims in (("slopes", slopes, torch.float32, 1), ("ranges", ranges, torch.int32, 2)):
            if t is None:
                continue
            if t.dtype != dtype or t.dim() != dims or not t.is_cuda or not t.is_contiguous() or (dims == 2 and t.shape[1] != 2):
                raise ValueError("slopes: fp32 [query_heads], ranges: int32 [total_tokens][2], contiguous CUDA tensors")
        given = [t for t in (slopes, ranges) if t is not None]
        if len({t.device for t in given}) > 1:
            raise ValueError("slopes and ranges of two devices")
        super().__init__(float(cap), None if slopes is None else slopes.data_ptr(), None if ranges is None else ranges.data_ptr())
        self.heads, self.rows = None if slopes is None else slopes.shape[0], None if ranges is None else ranges.shape[0]
        self.tensors, self.device_index = (slopes, ranges), given[0].device.index if given else -1

    def check(self, query_heads: int, total_tokens: int) -> None:
        if (self.heads is not None and self.heads < query_heads) or (self.rows is not None and self.rows < total_tokens):
            raise ValueError("a slope for every query head and a range for every token")


def paged_workspace(view: PagedView, batch: PagedBatch, query_heads: int, *, window: int = 0, sinks: int = 0, scoring: Optional[PagedScoring] = None, device=None) -> torch.Tensor:
    """Scratch for launch_paged_attention calls with this geometry and bounds no larger than the batch's (and with ranges, if the scoring has some)."""
    if scoring is None:
        n = int(lib.b200kv_paged_attn_workspace_bytes(C.byref(view), C.byref(batch), query_heads, window, sinks))
    else:
        n = int(lib.b200kv_paged_attn_scored_workspace_bytes(C.byref(view), C.byref(batch), C.byref(scoring), query_heads, window, sinks))
    return torch.empty(n, dtype=torch.uint8, device=device or "cuda")


def launch_paged_store(view: PagedView, batch: PagedBatch, key: torch.Tensor, value: torch.Tensor, k_norm_weight: Optional[torch.Tensor], *,
                       rope_mode: RopeMode = RopeMode.SECTIONED64, theta: float = 1.0e6, epsilon: float = 1.0e-6,
                       positions: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
    """launch_kv_store_quant for a ragged batch: key/value [total_tokens][kv_heads * head_dim] fp16 or fp32.  `positions` (int32
    [total_tokens]): what each token is rotated by where that is not its place in the cache."""
    rc = native.paged_store(view, batch, key, value, k_norm_weight, rope_mode, theta, epsilon, positions, stream)
    if rc:
        check(rc, "b200kv_paged_store")


def launch_paged_load(view: PagedView, batch: PagedBatch, key: Optional[torch.Tensor], value: Optional[torch.Tensor], *,
                      stream: Optional[torch.cuda.Stream] = None) -> None:
    """The rows of the batch's new tokens out of their pages, as fp16 [total_tokens][kv_heads][head_dim]; either side may be None."""
    rc = native.paged_load(view, batch, key, value, stream)
    if rc:
        check(rc, "b200kv_paged_load")


def launch_paged_attention(view: PagedView, batch: PagedBatch, q: torch.Tensor, output: torch.Tensor, *, query_heads: int, scale: float,
                           window: int = 0, sinks: int = 0, gate: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                           scoring: Optional[PagedScoring] = None, workspace: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Causal attention of every new token over its sequence's pages, times sigmoid(gate); with a window, over the last `window`
    positions and the first `sinks`.  q, output: fp16 or fp32 [total_tokens][query_heads][head_dim]; gate fp32; lse fp32
    [total_tokens][query_heads].  scoring: scores that are capped or biased, tokens that see otherwise.  workspace: `paged_workspace`."""
    if scoring is not None:
        scoring.check(query_heads, batch.total_tokens)
    rc = native.paged_attn(view, batch, query_heads, q, gate, output, lse, scale, window, sinks, workspace, stream, scoring)
    if rc:
        check(rc, "b200kv_paged_attn")


def launch_paged_weights(view: PagedView, batch: PagedBatch, q: torch.Tensor, lse: torch.Tensor, weights: torch.Tensor, *, query_heads: int,
                         scale: float, window: int = 0, sinks: int = 0, observe: int = 0, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Adds to `weights` (fp32 [sequences or more][kv_heads][max_length or more]) what the new tokens' attention gives each position, summed over
    tokens and heads; q, lse, scale, window and sinks of the attention call.  observe: only the last so many tokens of a sequence."""
    rc = native.paged_weights(view, batch, query_heads, q, lse, weights, scale, window, sinks, observe, stream)
    if rc:
        check(rc, "b200kv_paged_weights")


def launch_paged_evict(view: PagedView, batch: PagedBatch, target_table: torch.Tensor, weights: torch.Tensor, *, keep: int, sinks: int = 0,
                       recent: int = 0, kept: torch.Tensor, new_lengths: torch.Tensor, new_weights: Optional[torch.Tensor] = None,
                       stream: Optional[torch.cuda.Stream] = None) -> None:
    """Keeps the first `sinks`, the last `recent` and the heaviest other positions of every sequence and kv head, `keep` in all, moved together in the
    pages of target_table (int32 [sequences][pages]; the batch's own table: in place).  kept: int32 [sequences][kv_heads][keep],
    new_weights: fp32 of that shape, new_lengths: int32 [sequences].  Each may have rows for more sequences, which stay as they are."""
    rc = native.paged_evict(view, batch, keep, sinks, recent, target_table, weights, kept, new_weights, new_lengths, stream)
    if rc:
        check(rc, "b200kv_paged_evict")


class RotaryLayout(enum.IntEnum):
    """b200kv_rotary_layout: pairs (i, i + dims / 2) or (2i, 2i + 1)."""

    HALVES = 0
    NEIGHBOURS = 1


class RotaryScaling(enum.IntEnum):
    """b200kv_rotary_kind: how the frequencies are scaled for longer contexts."""

    NONE = 0
    LINEAR = 1
    BASE = 2
    BANDS = 3
    RAMP = 4


class RotaryTable(_lib.Rotary):
    """b200kv_rotary with its table on the device: the frequencies theta^(-2i / dims), scaled, or `frequencies` (radians a position, dims / 2 of them).

    factor: of every scaling; original_length, low, high: of BANDS and RAMP.  magnitude: what sines and cosines are multiplied by (the default: the scaling's own)."""

    def __init__(self, dims: int, *, theta: float = 1.0e6, layout: RotaryLayout = RotaryLayout.HALVES, scaling: RotaryScaling = RotaryScaling.NONE, factor: float = 1.0,
                 original_length: float = 0.0, low: float = 1.0, high: float = 32.0, frequencies: Optional[Sequence[float]] = None, magnitude: Optional[float] = None,
                 device: Optional[torch.device] = None):
        if not 0 < int(dims) <= 256 or int(dims) % 16:
            raise ValueError("dims: a multiple of 16 up to 256")
        turns, of_scaling = (C.c_uint64 * (dims // 2))(), C.c_float(1.0)
        if frequencies is not None:
            if len(frequencies) != dims // 2 or RotaryScaling(scaling) != RotaryScaling.NONE:
                raise ValueError("frequencies: one for every pair, as they are")
            check(lib.b200kv_rotary_turns_of((C.c_double * len(frequencies))(*map(float, frequencies)), len(frequencies), turns), "b200kv_rotary_turns_of")
        else:
            how = _lib.RotaryScaling(int(RotaryScaling(scaling)), factor, original_length, low, high)
            check(lib.b200kv_rotary_turns(dims, theta, C.byref(how), turns, C.byref(of_scaling)), "b200kv_rotary_turns")
        self.table = torch.frombuffer(bytearray(bytes(turns)), dtype=torch.int64).to(device or torch.device("cuda", torch.cuda.current_device()))
        super().__init__(self.table.data_ptr(), int(dims), int(RotaryLayout(layout)), of_scaling.value if magnitude is None else float(magnitude))
        self.device_index = self.table.device.index


def launch_paged_rotary(view: PagedView, batch: PagedBatch, rotary: RotaryTable, key: Optional[torch.Tensor], value: Optional[torch.Tensor], q: Optional[torch.Tensor] = None,
                        q_out: Optional[torch.Tensor] = None, *, query_heads: int = 0, gate: Optional[torch.Tensor] = None, q_norm_weight: Optional[torch.Tensor] = None,
                        k_norm_weight: Optional[torch.Tensor] = None, epsilon: float = 1.0e-6, positions: Optional[torch.Tensor] = None,
                        stream: Optional[torch.cuda.Stream] = None) -> None:
    """Norms and rotates a batch's queries and keys, and writes keys and values into their pages.  q [total_tokens][query_heads * head_dim], key and value [total_tokens]
    [kv_heads * head_dim]: fp16 or fp32, rows of any stride, such as columns of one matrix.  q_out: fp16 or fp32 [total_tokens][query_heads][head_dim], or q itself.  With gate (fp32
    [total_tokens][query_heads][head_dim]) a head of q is a query and its gate, and gate gets the second.  key and value may be None, or q and q_out."""
    if q is not None and query_heads <= 0:
        raise ValueError("query_heads is required with q")
    rc = native.paged_rotary(view, batch, rotary, query_heads, key, value, q, gate, q_out, q_norm_weight, k_norm_weight, epsilon, positions, stream)
    if rc:
        check(rc, "b200kv_paged_rotary")


class PageBook(_lib.PageBook):
    """b200kv_page_book over int32 CUDA tensors: refs [pages], tables [slots][max_pages], lengths [slots].  One book serves the pools of all layers; tables and lengths are what
    a PagedBatch takes."""

    def __init__(self, refs: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, *, page_size: int):
        if refs.dim() != 1 or tables.dim() != 2 or lengths.dim() != 1 or tables.shape[0] != lengths.shape[0]:
            raise ValueError("refs [pages], tables [slots][max_pages], lengths [slots]")
        for t in (refs, tables, lengths):
            if t.dtype != torch.int32 or not t.is_cuda or not t.is_contiguous() or t.device != refs.device:
                raise ValueError("expected contiguous int32 CUDA tensors of one device")
        super().__init__(refs.data_ptr(), tables.data_ptr(), lengths.data_ptr(), refs.numel(), int(page_size), lengths.numel(), tables.shape[1])
        self.tensors, self.device_index = (refs, tables, lengths), refs.device.index

    @classmethod
    def empty(cls, pages: int, page_size: int, slots: int, max_pages: int, device: Optional[torch.device] = None) -> "PageBook":
        dev = device or torch.device("cuda", torch.cuda.current_device())
        return cls(torch.zeros(pages, dtype=torch.int32, device=dev), torch.full((slots, max_pages), -1, dtype=torch.int32, device=dev),
                   torch.zeros(slots, dtype=torch.int32, device=dev), page_size=page_size)

    refs_tensor = property(lambda self: self.tensors[0])
    tables_tensor = property(lambda self: self.tensors[1])
    lengths_tensor = property(lambda self: self.tensors[2])


def pages_workspace(book: PageBook, device=None) -> torch.Tensor:
    """Scratch for launch_pages_* calls on this book."""
    n = int(lib.b200kv_pages_workspace_bytes(C.byref(book)))
    return torch.empty(n, dtype=torch.uint8, device=device or "cuda")


def launch_pages_grow(book: PageBook, slots: torch.Tensor, add: torch.Tensor, *, workspace: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Room for add[e] further positions of sequence slots[e] (int32 each, up to 8192 entries; a negative slot is left out): the lowest free pages, entry by entry."""
    rc = native.pages_grow(book, slots, add, workspace, stream)
    if rc:
        check(rc, "b200kv_pages_grow")


def launch_pages_fork(book: PageBook, views: Sequence[PagedView], parents: torch.Tensor, children: torch.Tensor, *, at: Optional[torch.Tensor] = None, workspace: torch.Tensor,
                      stream: Optional[torch.cuda.Stream] = None) -> None:
    """The empty slots children[e] go on from parents[e] (int32 each, as many entries at most as there are slots; a negative child is left out), with all its positions or the first
    at[e]: whole pages are shared, a last one that is not full is copied in the pools of all layers (`views`)."""
    rc = native.pages_fork(book, views, parents, children, at, workspace, stream)
    if rc:
        check(rc, "b200kv_pages_fork")


def launch_pages_free(book: PageBook, slots: torch.Tensor, *, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Sequences end: their slots (int32) become empty, their pages are given back."""
    rc = native.pages_free(book, slots, stream)
    if rc:
        check(rc, "b200kv_pages_free")


def launch_pages_compact(book: PageBook, views: Sequence[PagedView], moved: torch.Tensor, *, workspace: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Moves the pages that are held together at the front of the pools of all layers; moved (int32 [pages]): where each is now, -1 for one that was free."""
    rc = native.pages_compact(book, views, moved, workspace, stream)
    if rc:
        check(rc, "b200kv_pages_compact")


def launch_pages_copy(from_views: Sequence[PagedView], to_views: Sequence[PagedView], sources: torch.Tensor, targets: torch.Tensor, *,
                      stream: Optional[torch.cuda.Stream] = None) -> None:
    """Copies pages sources[i] of one set of pools to pages targets[i] of another of the same geometry (int32 each; a negative target: nothing)."""
    rc = native.pages_copy(from_views, to_views, sources, targets, stream)
    if rc:
        check(rc, "b200kv_pages_copy")

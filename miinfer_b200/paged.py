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
from typing import Optional

import torch

from . import _lib
from ._lib import check, lib, native
from .kv import KvCacheQuantMode, RopeMode

__all__ = ["PagedView", "PagedBatch", "PagedKvCache", "paged_workspace", "launch_paged_store", "launch_paged_load", "launch_paged_attention",
           "launch_paged_weights", "launch_paged_evict", "STATUS_BAD_PAGE", "STATUS_BAD_BOUND"]

STATUS_BAD_PAGE, STATUS_BAD_BOUND = 16, 32      # bits of the word registered with kv.set_status_word


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


def paged_workspace(view: PagedView, batch: PagedBatch, query_heads: int, *, window: int = 0, sinks: int = 0, device=None) -> torch.Tensor:
    """Scratch for launch_paged_attention calls with this geometry and bounds no larger than the batch's."""
    n = int(lib.b200kv_paged_attn_workspace_bytes(C.byref(view), C.byref(batch), query_heads, window, sinks))
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
                           workspace: torch.Tensor, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Causal attention of every new token over its sequence's pages, times sigmoid(gate); with a window, over the last `window`
    positions and the first `sinks`.  q, output: fp16 or fp32 [total_tokens][query_heads][head_dim]; gate fp32; lse fp32
    [total_tokens][query_heads].  workspace: `paged_workspace`."""
    rc = native.paged_attn(view, batch, query_heads, q, gate, output, lse, scale, window, sinks, workspace, stream)
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

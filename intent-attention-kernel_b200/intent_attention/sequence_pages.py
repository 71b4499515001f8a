"""Which sequences hold which pages of a pool: grow, fork, free and compact.

``SequencePages`` is the bookkeeping of one layer's pages on the GPU: a count of
holders per page (0 = free), the page table of every slot and table head, and
the tokens of every slot.  Its ``table`` and ``lengths`` are what the attention
and append calls take.  Sequences share pages after ``fork_sequences``; a shared
page that is part full is copied by ``grow_sequences`` before its holder writes
into it.  Pages of ``PagePool`` and ``Fp4Pool`` alike.

All operations run on the device without reading anything back, are exact and
do not depend on the order in which blocks run; ``rejected`` (an int32 CUDA
counter, optional) collects what they refuse.  A pool's operations follow one
another on one stream.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Union

import torch

from . import _native as N
from .fp4_cache import Fp4Pool, _index_tensor, _on
from .paged import PagePool, _ptr, _require_cuda, _stream, _tags_args

_BIT = {f: 1 << getattr(N, f"FMT_{f}") for f in ("F16", "FP8", "INT8", "INT4", "INT4R")}
_SCALED = _BIT["FP8"] | _BIT["INT8"] | _BIT["INT4"] | _BIT["INT4R"]
_PLANE_FORMATS = {"f16": _BIT["F16"], "fp8": _BIT["FP8"], "i8": _BIT["INT8"], "i4": _BIT["INT4"] | _BIT["INT4R"],
                  "i4r": _BIT["INT4R"], "scale": _SCALED, "res_scale": _BIT["INT4R"]}


@dataclass
class SequencePages:
    """``refs`` int32 [num_pages], ``table`` int32 [slots, Ht, W], ``lengths`` int32 [slots], all on one device."""

    refs: torch.Tensor
    table: torch.Tensor
    lengths: torch.Tensor
    page_size: int

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, num_slots: int, table_heads: int, width: int,
                 device="cuda") -> "SequencePages":
        """Every page free, every slot empty."""
        dev = torch.device(device)
        return cls(torch.zeros(num_pages, dtype=torch.int32, device=dev),
                   torch.full((num_slots, table_heads, width), -1, dtype=torch.int32, device=dev),
                   torch.zeros(num_slots, dtype=torch.int32, device=dev), page_size)

    def struct(self) -> N.SeqPages:
        dev = self.refs.device
        _index_tensor(self.refs, "refs", dev)
        _index_tensor(self.lengths, "lengths", dev)
        _require_cuda(self.table, "table")
        t = self.table
        if t.device != dev or t.dtype != torch.int32 or t.dim() != 3 or (t.stride(2) != 1 and t.shape[2] > 1):
            raise ValueError(f"table must be int32 [slots, Ht, W] with contiguous rows on {dev}")
        if self.lengths.numel() != t.shape[0]:
            raise ValueError(f"lengths must have {t.shape[0]} entries, got {self.lengths.numel()}")
        if self.page_size <= 0:
            raise ValueError("page_size must be positive")
        s = N.SeqPages()
        s.refs, s.num_pages = self.refs.data_ptr(), self.refs.numel()
        s.page_table, s.pt_stride_s, s.pt_stride_h, s.table_width = t.data_ptr(), t.stride(0), t.stride(1), t.shape[2]
        s.lengths, s.num_slots, s.num_table_heads = self.lengths.data_ptr(), t.shape[0], t.shape[1]
        s.page_size = self.page_size
        return s


def _planes(pool: Union[PagePool, Fp4Pool], pages: SequencePages, page_tags, tag_map, tag_default) -> N.PagePlanes:
    if pool.num_pages != pages.refs.numel() or pool.page_size != pages.page_size:
        raise ValueError(f"pages count {pages.refs.numel()} pages of {pages.page_size} rows, the pool has "
                         f"{pool.num_pages} of {pool.page_size}")
    if isinstance(pool, Fp4Pool):
        pool.struct()                         # checks the planes
        named = [(t, 0) for t in pool.tensors()]
    else:
        named = [(getattr(pool, f"{side}_{n}"), f) for n, f in _PLANE_FORMATS.items() for side in ("k", "v")]
        named = [(t, f) for t, f in named if t is not None]
    s = N.PagePlanes()
    for i, (t, formats) in enumerate(named):
        _require_cuda(t, "page pool")
        if t.device != pages.refs.device:
            raise ValueError(f"the pool is on {t.device}, its pages on {pages.refs.device}")
        if not t.is_contiguous() or t.shape[0] != pool.num_pages:
            raise ValueError("page pools must be contiguous [num_pages, ...] tensors")
        if t.numel():
            s.base[i], s.bytes[i], s.formats[i] = t.data_ptr(), t.numel() // pool.num_pages * t.element_size(), formats
            s.num_planes = i + 1
    if page_tags is not None:
        if isinstance(pool, Fp4Pool):
            raise ValueError("an Fp4Pool has one format: no page_tags")
        if tag_map is None:
            raise ValueError("page_tags needs a tag_map")
        s.page_tags, s.tag_bytes = _tags_args(page_tags)
        if page_tags.numel() < pool.num_pages or page_tags.device != pages.refs.device:
            raise ValueError(f"page_tags must hold {pool.num_pages} tags on {pages.refs.device}")
        for i, f in enumerate(tag_map):
            s.tag_map[i] = f
        s.tag_default = tag_default
    return s


def _workspace(pages: SequencePages, s: N.SeqPages) -> torch.Tensor:
    n = ctypes.c_size_t(0)
    N.check(N.lib().iak_pages_workspace_size(ctypes.byref(s), ctypes.byref(n)), "iak_pages_workspace_size")
    # of this call alone, as calls captured into different graphs must not share it
    return torch.empty(n.value, dtype=torch.uint8, device=pages.refs.device)


def grow_sequences(pool: Union[PagePool, Fp4Pool], pages: SequencePages, new_tokens: torch.Tensor,
                   rejected: Optional[torch.Tensor] = None, page_tags: Optional[torch.Tensor] = None,
                   tag_map: Optional[Sequence[int]] = None, tag_default: int = N.FMT_SKIP) -> None:
    """Make room for ``new_tokens[s]`` (int32 [slots]) more tokens of every slot and add them to its length.

    Fresh pages are the lowest free ones, given out in order of (slot, head,
    table entry).  A slot that gets tokens while its last page is part full and
    held by others too first gets a copy of that page (all planes of the
    pool; with ``page_tags`` and ``tag_map`` those of the page's format, and its
    tag).  The tokens themselves are the caller's to write.  Refused: a
    negative count; tokens beyond the table's width; an open page outside the
    pool; and, once the free pages run out, the first slot that does not fit and
    every later one that gets tokens.
    """
    s = pages.struct()
    _index_tensor(new_tokens, "new_tokens", pages.refs.device, pages.table.shape[0])
    _index_tensor(rejected, "rejected", pages.refs.device, 1)
    pl = _planes(pool, pages, page_tags, tag_map, tag_default)
    with _on(pages.refs.device):
        ws = _workspace(pages, s)
        N.check(N.lib().iak_pages_grow(ctypes.byref(s), ctypes.byref(pl), new_tokens.data_ptr(), _ptr(rejected),
                                       ws.data_ptr(), ws.numel(), _stream(pages.refs.device)), "iak_pages_grow")


def fork_sequences(pages: SequencePages, src: torch.Tensor, dst: torch.Tensor,
                   rejected: Optional[torch.Tensor] = None) -> None:
    """Slot ``dst[i]`` becomes a copy of ``src[i]`` that shares all of its pages (int32 lists on the device).

    Refused: a slot out of range, a dst that holds tokens, a dst listed before,
    a src that is also a dst of the call.
    """
    s = pages.struct()
    _index_tensor(src, "src", pages.refs.device)
    _index_tensor(dst, "dst", pages.refs.device, src.numel())
    _index_tensor(rejected, "rejected", pages.refs.device, 1)
    with _on(pages.refs.device):
        N.check(N.lib().iak_pages_fork(ctypes.byref(s), src.data_ptr(), dst.data_ptr(), src.numel(), _ptr(rejected),
                                       _stream(pages.refs.device)), "iak_pages_fork")


def free_sequences(pages: SequencePages, slots: torch.Tensor, rejected: Optional[torch.Tensor] = None) -> None:
    """The listed slots (int32 on the device) let go of their pages: table entries -1, length 0.  A slot listed
    twice is freed once; one out of range is refused."""
    s = pages.struct()
    _index_tensor(slots, "slots", pages.refs.device)
    _index_tensor(rejected, "rejected", pages.refs.device, 1)
    with _on(pages.refs.device):
        N.check(N.lib().iak_pages_free(ctypes.byref(s), slots.data_ptr(), slots.numel(), _ptr(rejected),
                                       _stream(pages.refs.device)), "iak_pages_free")


def compact_pages(pool: Union[PagePool, Fp4Pool], pages: SequencePages, page_tags: Optional[torch.Tensor] = None,
                  tag_map: Optional[Sequence[int]] = None, tag_default: int = N.FMT_SKIP) -> torch.Tensor:
    """Pack the n pages in use into pages 0 .. n - 1 and return n (int32, 0-d, on the device).

    Pages in use at or above n move to the free pages below n, both in ascending
    order; tables and counts follow.  With ``page_tags`` and ``tag_map`` only the
    planes of each page's format move, and its tag.
    """
    s = pages.struct()
    pl = _planes(pool, pages, page_tags, tag_map, tag_default)
    live = torch.empty((), dtype=torch.int32, device=pages.refs.device)
    with _on(pages.refs.device):
        ws = _workspace(pages, s)
        N.check(N.lib().iak_pages_compact(ctypes.byref(s), ctypes.byref(pl), live.data_ptr(), ws.data_ptr(),
                                          ws.numel(), _stream(pages.refs.device)), "iak_pages_compact")
    return live

"""Which sequences hold which pages of a pool: grow, shrink, fork, free and compact.

``SequencePages`` is the bookkeeping of one layer's pages on the GPU: a count of
holders per page (0 = free), the page table of every slot and table head, and
the tokens of every slot.  Its ``table`` and ``lengths`` are what the attention
and append calls take.  Sequences share pages after ``fork_sequences``; a shared
page that is part full is copied by ``grow_sequences`` before its holder writes
into it.  A step of a serving loop::

    start = pages.lengths.clone()
    grow_sequences(pool, pages, new_tokens)
    got = pages.lengths - start
    append_fp4(pool, k_new, v_new, pages.table, start, got)

``got`` is 0 for the slots that were refused (no free page, a full table):
rows written for them all the same would land in an open page that other
sequences may still share.  Their outputs of the step are over the old tokens.

The operations copy and move pages of ``PagePool`` and ``Fp4Pool`` alike, but
only ``Fp4Pool``'s calls follow a table and lengths.  ``append_tokens`` and
``route_pages`` name a ``PagePool``'s pages by ``bases`` (those of a sequence
lie together, the open one staged in ``KVStage``) and do not apply to pages
that these operations hand out: write such pages with ``PagePool.quantize_``
and attend to whole pages by table and page counts (``paged_decode``).

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
from .fp4_cache import Fp4Pool, _check_device, _index_tensor, _on, _page_table, _raw_stream
from .paged import PagePool, _require_cuda, _tags_args

_BIT = {f: 1 << getattr(N, f"FMT_{f}") for f in ("F16", "FP8", "INT8", "INT4", "INT4R")}
_SCALED = _BIT["FP8"] | _BIT["INT8"] | _BIT["INT4"] | _BIT["INT4R"]
# a PagePool's planes and the formats of the pages that use them
_PLANES = tuple((f"{side}_{name}", bits) for name, bits in (
    ("f16", _BIT["F16"]), ("fp8", _BIT["FP8"]), ("i8", _BIT["INT8"]), ("i4", _BIT["INT4"] | _BIT["INT4R"]),
    ("i4r", _BIT["INT4R"]), ("scale", _SCALED), ("res_scale", _BIT["INT4R"])) for side in "kv")


@dataclass
class SequencePages:
    """``refs`` int32 [num_pages], ``table`` int32 [slots, Ht, W], ``lengths`` int32 [slots], all on one device.
    The table may be a view with strides; its rows are contiguous and do not overlap."""

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
        _require_cuda(self.refs, "refs")
        dev = self.refs.get_device()
        if self.page_size <= 0:
            raise ValueError("page_size must be positive")
        pt, ss, sh, Ht, W = _page_table(self.table, dev)
        slots = self.table.shape[0]
        # every entry is written on its own: rows one after another, slots or heads outermost
        inner, outer = ((sh, Ht), (ss, slots)) if ss >= sh else ((ss, slots), (sh, Ht))
        row = W if inner[1] <= 1 else W + (inner[1] - 1) * inner[0]
        if (inner[1] > 1 and inner[0] < W) or (outer[1] > 1 and outer[0] < row):
            raise ValueError("table rows must not overlap (an expanded view?)")
        return N.SeqPages(_index_tensor(self.refs, "refs", dev), self.refs.numel(), pt, ss, sh, W,
                          _index_tensor(self.lengths, "lengths", dev, slots), slots, Ht, self.page_size)


def _planes(pool: Union[PagePool, Fp4Pool], pages: SequencePages, page_tags, tag_map, tag_default) -> N.PagePlanes:
    if pool.num_pages != pages.refs.numel() or pool.page_size != pages.page_size:
        raise ValueError(f"pages count {pages.refs.numel()} pages of {pages.page_size} rows, the pool has "
                         f"{pool.num_pages} of {pool.page_size}")
    dev = pages.refs.get_device()
    if isinstance(pool, Fp4Pool):
        planes = ((pool.data, 0),)
    else:
        planes = [(t, f) for t, f in [(getattr(pool, name), f) for name, f in _PLANES] if t is not None]
    s = N.PagePlanes()
    base, sizes, formats = s.base, s.bytes, s.formats
    n = 0
    for t, f in planes:
        _check_device(t, "page pool", dev)
        if not t.is_contiguous() or t.shape[0] != pool.num_pages:
            raise ValueError("page pools must be contiguous [num_pages, ...] tensors")
        size = t.nbytes
        if size:
            base[n], sizes[n], formats[n] = t.data_ptr(), size // pool.num_pages, f
            n += 1
    s.num_planes = n
    if page_tags is not None:
        if isinstance(pool, Fp4Pool):
            raise ValueError("an Fp4Pool has one format: no page_tags")
        if tag_map is None:
            raise ValueError("page_tags needs a tag_map")
        s.page_tags, s.tag_bytes = _tags_args(page_tags)
        _check_device(page_tags, "page_tags", dev)
        if page_tags.numel() < pool.num_pages:
            raise ValueError(f"page_tags must hold {pool.num_pages} tags")
        for i, f in enumerate(tag_map):
            s.tag_map[i] = f
        s.tag_default = tag_default
    return s


def _workspace(device: torch.device, s: N.SeqPages) -> torch.Tensor:
    n = ctypes.c_size_t(0)
    N.check(N.lib().iak_pages_workspace_size(ctypes.byref(s), ctypes.byref(n)), "iak_pages_workspace_size")
    # of this call alone, as calls captured into different graphs must not share it
    return torch.empty(n.value, dtype=torch.uint8, device=device)


def grow_sequences(pool: Union[PagePool, Fp4Pool], pages: SequencePages, new_tokens: torch.Tensor,
                   rejected: Optional[torch.Tensor] = None, page_tags: Optional[torch.Tensor] = None,
                   tag_map: Optional[Sequence[int]] = None, tag_default: int = N.FMT_SKIP) -> None:
    """Make room for ``new_tokens[s]`` (int32 [slots]) more tokens of every slot and add them to its length.

    Fresh pages are the lowest free ones, given out in order of (slot, head,
    table entry).  A slot that gets tokens while its last page is part full and
    held by others too first gets a copy of that page (all planes of the
    pool; with ``page_tags`` and ``tag_map`` those of the page's format, and its
    tag).  The tokens themselves are the caller's to write, for slots whose
    length has grown.  Refused: a
    negative count; tokens beyond the table's width; an open page outside the
    pool; and, once the free pages run out, the first slot that does not fit and
    every later one that gets tokens.
    """
    s = pages.struct()
    dev = pages.refs.get_device()
    more = _index_tensor(new_tokens, "new_tokens", dev, s.num_slots)
    count = _index_tensor(rejected, "rejected", dev, 1)
    pl = _planes(pool, pages, page_tags, tag_map, tag_default)
    with _on(dev):
        ws = _workspace(pages.refs.device, s)
        N.check(N.lib().iak_pages_grow(ctypes.byref(s), ctypes.byref(pl), more, count, ws.data_ptr(), ws.numel(),
                                       _raw_stream(dev)), "iak_pages_grow")


def shrink_sequences(pages: SequencePages, tokens: torch.Tensor, rejected: Optional[torch.Tensor] = None) -> None:
    """Take ``tokens[s]`` (int32 [slots]) tokens off the end of every slot, as when draft tokens are not kept; pages
    that are left without a token of the slot are let go of.  Refused: a negative count, more than the slot holds.

    Lengths must not be lowered in any other way: the pages left behind would never be free again.
    """
    s = pages.struct()
    dev = pages.refs.get_device()
    a = _index_tensor(tokens, "tokens", dev, s.num_slots)
    count = _index_tensor(rejected, "rejected", dev, 1)
    with _on(dev):
        N.check(N.lib().iak_pages_shrink(ctypes.byref(s), a, count, _raw_stream(dev)), "iak_pages_shrink")


def fork_sequences(pages: SequencePages, src: torch.Tensor, dst: torch.Tensor,
                   rejected: Optional[torch.Tensor] = None) -> None:
    """Slot ``dst[i]`` becomes a copy of ``src[i]`` that shares all of its pages (int32 lists on the device).

    Refused: a slot out of range, a dst that holds tokens, a dst listed before,
    a src that is also a dst of the call.
    """
    s = pages.struct()
    dev = pages.refs.get_device()
    a, n = _index_tensor(src, "src", dev), src.numel()
    b = _index_tensor(dst, "dst", dev, n)
    count = _index_tensor(rejected, "rejected", dev, 1)
    with _on(dev):
        N.check(N.lib().iak_pages_fork(ctypes.byref(s), a, b, n, count, _raw_stream(dev)), "iak_pages_fork")


def free_sequences(pages: SequencePages, slots: torch.Tensor, rejected: Optional[torch.Tensor] = None) -> None:
    """The listed slots (int32 on the device) let go of their pages: table entries -1, length 0.  A slot listed
    twice is freed once; one out of range is refused."""
    s = pages.struct()
    dev = pages.refs.get_device()
    a = _index_tensor(slots, "slots", dev)
    count = _index_tensor(rejected, "rejected", dev, 1)
    with _on(dev):
        N.check(N.lib().iak_pages_free(ctypes.byref(s), a, slots.numel(), count, _raw_stream(dev)), "iak_pages_free")


def compact_pages(pool: Union[PagePool, Fp4Pool], pages: SequencePages, page_tags: Optional[torch.Tensor] = None,
                  tag_map: Optional[Sequence[int]] = None, tag_default: int = N.FMT_SKIP) -> torch.Tensor:
    """Pack the n pages in use into pages 0 .. n - 1 and return n (int32, 0-d, on the device).

    Pages in use at or above n move to the free pages below n, both in ascending
    order; tables and counts follow.  With ``page_tags`` and ``tag_map`` only the
    planes of each page's format move, and its tag.
    """
    s = pages.struct()
    dev = pages.refs.get_device()
    pl = _planes(pool, pages, page_tags, tag_map, tag_default)
    live = torch.empty((), dtype=torch.int32, device=pages.refs.device)
    with _on(dev):
        ws = _workspace(pages.refs.device, s)
        N.check(N.lib().iak_pages_compact(ctypes.byref(s), ctypes.byref(pl), live.data_ptr(), ws.data_ptr(),
                                          ws.numel(), _raw_stream(dev)), "iak_pages_compact")
    return live

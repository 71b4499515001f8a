"""A paged KV cache in 4-bit floating point and the attention that reads it.

``Fp4Pool`` holds K and V rows as E2M1 codes with one power-of-two scale per
row and 32 channels (4.25 bits an element).  A row is quantised once, when it is
written: appending needs no staged copy of the open page, and what a cached
token stands for never changes afterwards.  Pages are single-head, as in
``PagePool``; token t of (sequence b, table head h) is row ``t % page_size`` of
page ``page_table[b, h, t // page_size]``.

A value x of a block becomes the E2M1 value (0, 0.5, 1, 1.5, 2, 3, 4, 6) nearest
to x * 2^-e, ties to the even code, where e is the smallest integer with
6 * 2^e >= the block's largest magnitude, held in [-14, 13].  Magnitudes above
6 * 2^13 = 49152 become 49152, NaN becomes 0; blocks below 2^-16 become 0.

No call synchronises or reads device data on the host; all of them can be
captured into CUDA graphs.  Index tensors are int32 on the pool's device.
"""

from __future__ import annotations

import contextlib
import ctypes
import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _native as N
from .paged import _DT, _ptr, _require_cuda, _stream

HEAD_DIMS = (64, 128, 256)


def _on(device: torch.device):
    """The library launches on the current device; switch only when it is another one."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _index_tensor(t: Optional[torch.Tensor], name: str, device: torch.device, numel: Optional[int] = None):
    """An int32 vector on ``device`` with unit stride; None passes."""
    if t is None:
        return None
    _require_cuda(t, name)
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the pool on {device}")
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must have {numel} entries, got {t.numel()}")
    return t


def _page_table(page_table: torch.Tensor, device: torch.device, batch: Optional[int] = None,
                heads: Optional[int] = None) -> torch.Tensor:
    _require_cuda(page_table, "page_table")
    if page_table.device != device:
        raise ValueError(f"page_table is on {page_table.device}, the pool on {device}")
    if page_table.dim() != 3 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [B, Ht, W]")
    if page_table.stride(2) != 1 and page_table.shape[2] > 1:
        raise ValueError("page_table rows must be contiguous")
    if (batch is not None and page_table.shape[0] != batch) or (heads is not None and page_table.shape[1] != heads):
        raise ValueError(f"page_table must be [{batch}, {heads if heads is not None else 'Ht'}, W], "
                         f"got {tuple(page_table.shape)}")
    return page_table


@dataclass
class Fp4Pool:
    """K/V pages of one layer on one device in 4-bit floating point.

    The byte order inside a page is the kernels' own (``include/intent_attention_b200.h``);
    ``append_fp4`` writes it and ``read_fp4`` reads it back.
    """

    num_pages: int
    page_size: int
    head_dim: int
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, head_dim: int, device="cuda", zero: bool = False) -> "Fp4Pool":
        """A pool of ``num_pages`` pages; ``zero`` clears the codes too (the scales always start at 0)."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size must be a positive multiple of 16, got {page_size}")
        if num_pages < 0:
            raise ValueError("num_pages must not be negative")
        dev = torch.device(device)
        codes, scales = (num_pages, page_size, head_dim // 2), (num_pages, page_size, head_dim // 32)
        mk = torch.zeros if zero else torch.empty
        return cls(num_pages, page_size, head_dim,
                   mk(codes, dtype=torch.uint8, device=dev), torch.zeros(scales, dtype=torch.uint8, device=dev),
                   mk(codes, dtype=torch.uint8, device=dev), torch.zeros(scales, dtype=torch.uint8, device=dev))

    @property
    def device(self) -> torch.device:
        return self.k_codes.device

    def tensors(self):
        return [self.k_codes, self.k_scales, self.v_codes, self.v_scales]

    def nbytes(self) -> int:
        return sum(t.numel() for t in self.tensors())

    def struct(self) -> N.Fp4PoolStruct:
        s = N.Fp4PoolStruct()
        rows = self.num_pages * self.page_size
        for name, t, per in (("k_codes", self.k_codes, 2), ("k_scales", self.k_scales, 32),
                             ("v_codes", self.v_codes, 2), ("v_scales", self.v_scales, 32)):
            _require_cuda(t, name)
            if t.device != self.device:
                raise ValueError("the pool's planes lie on different devices")
            if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != rows * (self.head_dim // per):
                raise ValueError(f"{name} must be contiguous uint8 of {rows * (self.head_dim // per)} bytes")
            setattr(s, name, t.data_ptr())
        s.num_pages, s.page_size, s.head_dim = self.num_pages, self.page_size, self.head_dim
        return s


# ---------------------------------------------------------------------- #
#  Rows in and out
# ---------------------------------------------------------------------- #

def _rows_args(pool: Fp4Pool, k, v, page_table, positions, counts) -> N.Fp4RowsArgs:
    B, Ht, n, _ = k.shape
    a = N.Fp4RowsArgs()
    a.k, a.v, a.dtype = k.data_ptr(), v.data_ptr(), _DT[k.dtype]
    a.k_stride_b, a.k_stride_h, a.k_stride_n = k.stride(0), k.stride(1), k.stride(2)
    a.v_stride_b, a.v_stride_h, a.v_stride_n = v.stride(0), v.stride(1), v.stride(2)
    a.batch, a.num_table_heads, a.num_rows = B, Ht, n
    pt = _page_table(page_table, pool.device, B, Ht)
    a.page_table, a.pt_stride_b, a.pt_stride_h, a.table_width = pt.data_ptr(), pt.stride(0), pt.stride(1), pt.shape[2]
    a.positions = _ptr(_index_tensor(positions, "positions", pool.device, B))
    a.counts = _ptr(_index_tensor(counts, "counts", pool.device, B))
    return a


def append_fp4(pool: Fp4Pool, k_new: torch.Tensor, v_new: torch.Tensor, page_table: torch.Tensor,
               positions: Optional[torch.Tensor] = None, counts: Optional[torch.Tensor] = None,
               dropped: Optional[torch.Tensor] = None) -> None:
    """Quantise ``k_new`` / ``v_new`` [B, Ht, n, D] (float32 / float16 / bfloat16, any strides with a
    unit last one) into the pool.

    Row i of sequence b is its token ``positions[b] + i`` (``positions`` None =
    0); rows from ``counts[b]`` on (a padded batch; None = none) are not
    written.  Rows whose table slot or page does not exist are left out and
    added to ``dropped`` (an int32 CUDA counter).  The pages written in one call
    belong to one (b, h) each, and a sequence is written by one call at a time:
    two rows of V share their bytes.
    """
    for name, x in (("k_new", k_new), ("v_new", v_new)):
        _require_cuda(x, name)
        if x.device != pool.device:
            raise ValueError(f"{name} is on {x.device}, the pool on {pool.device}")
    if k_new.dim() != 4 or k_new.shape != v_new.shape or k_new.shape[3] != pool.head_dim:
        raise ValueError(f"k_new / v_new must both be [B, Ht, n, {pool.head_dim}]")
    if k_new.dtype != v_new.dtype or k_new.dtype not in _DT:
        raise ValueError("k_new / v_new must share a float32 / float16 / bfloat16 dtype")
    if k_new.stride(3) != 1:
        k_new = k_new.contiguous()
    if v_new.stride(3) != 1:
        v_new = v_new.contiguous()
    a = _rows_args(pool, k_new, v_new, page_table, positions, counts)
    a.dropped = _ptr(_index_tensor(dropped, "dropped", pool.device, 1))
    s = pool.struct()
    with _on(pool.device):
        N.check(N.lib().iak_fp4_append(ctypes.byref(s), ctypes.byref(a), _stream(pool.device)), "iak_fp4_append")


def read_fp4(pool: Fp4Pool, page_table: torch.Tensor, positions: Optional[torch.Tensor], num_rows: int,
             counts: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached tokens ``positions[b] .. positions[b] + num_rows - 1`` as dense (k, v)
    [B, Ht, num_rows, D].  Every value a pool holds is exact in all three float
    types.  Rows from ``counts[b]`` on, and rows of slots or pages that do not
    exist, are 0.  ``out``: a (k, v) pair to write into."""
    _page_table(page_table, pool.device)
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    shape = (page_table.shape[0], page_table.shape[1], num_rows, pool.head_dim)
    if out is None:
        if dtype not in _DT:
            raise ValueError("dtype must be float32 / float16 / bfloat16")
        k, v = (torch.empty(shape, dtype=dtype, device=pool.device) for _ in range(2))
    else:
        k, v = out
        for name, x in (("out[0]", k), ("out[1]", v)):
            _require_cuda(x, name)
            if tuple(x.shape) != shape or x.device != pool.device or x.dtype not in _DT or x.dtype != k.dtype:
                raise ValueError(f"{name} must be a {shape} float tensor on {pool.device}, both of one dtype")
            if x.stride(3) != 1:
                raise ValueError(f"{name} needs a unit stride along head_dim")
    a = _rows_args(pool, k, v, page_table, positions, counts)
    s = pool.struct()
    with _on(pool.device):
        N.check(N.lib().iak_fp4_read(ctypes.byref(s), ctypes.byref(a), _stream(pool.device)), "iak_fp4_read")
    return k, v


# ---------------------------------------------------------------------- #
#  Attention
# ---------------------------------------------------------------------- #

def _decode(q: torch.Tensor, pool: Fp4Pool, page_table: torch.Tensor, lengths: torch.Tensor, sm_scale: float,
            out: Optional[torch.Tensor], out_dtype: Optional[torch.dtype], differential=None) -> torch.Tensor:
    _require_cuda(q, "q")
    dev = pool.device
    if q.device != dev:
        raise ValueError(f"q is on {q.device}, the pool on {dev}")
    if q.dim() not in (3, 4) or q.shape[-1] != pool.head_dim:
        raise ValueError(f"q must be [B, Hq, {pool.head_dim}] or [B, Hq, M, {pool.head_dim}], got {tuple(q.shape)}")
    if q.dtype not in _DT:
        raise ValueError(f"q dtype {q.dtype} unsupported")
    if q.stride(-1) != 1:
        q = q.contiguous()
    B, Hq = q.shape[0], q.shape[1]
    M = q.shape[2] if q.dim() == 4 else 1
    if M > N.FP4_MAX_QUERIES:
        raise ValueError(f"at most {N.FP4_MAX_QUERIES} queries per sequence, got {M}: read_fp4 the context for a prompt")
    pt = _page_table(page_table, dev, B)
    Ht = pt.shape[1]
    if Hq and (Ht == 0 or Hq % Ht):
        raise ValueError(f"query heads ({Hq}) must be a multiple of page-table heads ({Ht})")
    if lengths is None:
        raise ValueError("lengths [B] is required")
    _index_tensor(lengths, "lengths", dev, B)
    if out is None:
        out = torch.empty(q.shape, dtype=out_dtype or q.dtype, device=dev)
    _require_cuda(out, "out")
    if out.shape != q.shape or out.device != dev or out.dtype not in _DT or out.stride(-1) != 1:
        raise ValueError(f"out must be a {tuple(q.shape)} float tensor on {dev} with a contiguous last dim")
    a = N.Fp4DecodeArgs()
    a.q, a.q_dtype, a.q_stride_b, a.q_stride_h = q.data_ptr(), _DT[q.dtype], q.stride(0), q.stride(1)
    a.out, a.out_dtype, a.out_stride_b, a.out_stride_h = out.data_ptr(), _DT[out.dtype], out.stride(0), out.stride(1)
    if q.dim() == 4:
        a.q_stride_m, a.out_stride_m = q.stride(2), out.stride(2)
    a.batch, a.num_q_heads, a.num_table_heads, a.num_queries = B, Hq, Ht, M
    a.page_table, a.pt_stride_b, a.pt_stride_h, a.table_width = pt.data_ptr(), pt.stride(0), pt.stride(1), pt.shape[2]
    a.lengths, a.sm_scale = lengths.data_ptr(), sm_scale
    if differential is not None:
        lam, norm_weight, eps, out_scale = differential
        a.differential, a.lam, a.norm_weight = 1, lam.data_ptr(), _ptr(norm_weight)
        a.eps, a.out_scale = eps, out_scale
    s = pool.struct()
    L = N.lib()
    nbytes = ctypes.c_size_t(0)
    with _on(dev):
        N.check(L.iak_fp4_decode_workspace_size(ctypes.byref(s), ctypes.byref(a), ctypes.byref(nbytes)),
                "iak_fp4_decode_workspace_size")
        # of this call alone: calls on other streams, or captured into other graphs, never share it
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=dev) if nbytes.value else None
        N.check(L.iak_fp4_decode(ctypes.byref(s), ctypes.byref(a), _ptr(ws), nbytes.value, _stream(dev)),
                "iak_fp4_decode")
    return out


def paged_decode_fp4(q: torch.Tensor, pool: Fp4Pool, page_table: torch.Tensor, lengths: torch.Tensor,
                     sm_scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                     out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """softmax(sm_scale q K') V over each sequence's ``lengths[b]`` cached tokens.

    ``q`` [B, Hq, D] is one token per sequence; [B, Hq, M, D] are its last M
    tokens (M <= 16, draft tokens checked together), of which query m sees the
    tokens before ``lengths[b] - (M - 1 - m)``.  Query head h reads table head
    h // (Hq // Ht).  Lengths beyond the table count as its capacity; pages
    outside the pool are not seen; a query that sees no token gives 0.
    ``sm_scale`` defaults to 1 / sqrt(D).
    """
    scale = 1.0 / math.sqrt(pool.head_dim) if sm_scale is None else float(sm_scale)
    return _decode(q, pool, page_table, lengths, scale, out, out_dtype)


def differential_decode_fp4(q: torch.Tensor, pool: Fp4Pool, page_table: torch.Tensor, lengths: torch.Tensor,
                            lam: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                            out_scale: float = 1.0, sm_scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None,
                            out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """Differential attention over the same cache, the last step of a layer fused in.

    The two halves of a query and of a K row make two softmax maps over the
    same V rows:  x = (softmax(sm_scale q1 K1') - lam[head] softmax(sm_scale q2 K2')) V.
    ``lam`` float32 [Hq] are the learned weights.  The output is out_scale * x,
    or with ``norm_weight`` (float32 [D]) out_scale * norm_weight * x /
    sqrt(mean(x^2) + eps) over each head's D channels.  ``sm_scale`` defaults to
    1 / sqrt(D / 2).  Everything else as in ``paged_decode_fp4``.
    """
    def weight(t, name, n):
        _require_cuda(t, name)
        if t.device != pool.device or t.dtype != torch.float32 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous float32 values on {pool.device}")
        return t

    if not isinstance(q, torch.Tensor) or q.dim() < 2:
        raise ValueError("q must be [B, Hq, D] or [B, Hq, M, D]")
    weight(lam, "lam", q.shape[1])
    if norm_weight is not None:
        weight(norm_weight, "norm_weight", pool.head_dim)
    if not (eps >= 0.0 and math.isfinite(eps) and math.isfinite(out_scale)):
        raise ValueError("eps must be finite and not negative, out_scale finite")
    scale = 1.0 / math.sqrt(pool.head_dim // 2) if sm_scale is None else float(sm_scale)
    return _decode(q, pool, page_table, lengths, scale, out, out_dtype, (lam, norm_weight, float(eps), float(out_scale)))

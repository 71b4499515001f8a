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
from .paged import _DT, _require_cuda

HEAD_DIMS = (64, 128, 256)

# Per-call host work is most of a small call's time: the helpers below take the device as its index (a CPU tensor's is
# -1), test the few properties that the kernels rely on and build their messages only when one fails.
_NO_SWITCH = contextlib.nullcontext()


def _on(dev: int):
    """The library launches on the current device; switch only when it is another one."""
    return _NO_SWITCH if dev == torch._C._cuda_getDevice() else torch.cuda.device(dev)


def _raw_stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)        # (a torch build without CUDA lacks the name: not at import)


def _check_device(t, name: str, dev: int) -> None:
    if not isinstance(t, torch.Tensor) or t.get_device() != dev:
        _require_cuda(t, name)
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")


def _index_tensor(t: Optional[torch.Tensor], name: str, dev: int, numel: Optional[int] = None):
    """Address of a contiguous int32 tensor on device ``dev``; None passes."""
    if t is None:
        return None
    _check_device(t, name, dev)
    if t.dtype is not torch.int32 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor")
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} must have {numel} entries, got {t.numel()}")
    return t.data_ptr()


def _page_table(t: torch.Tensor, dev: int, batch: Optional[int] = None, heads: Optional[int] = None):
    """(address, stride of b, stride of h, Ht, W) of an int32 [B, Ht, W] table."""
    _check_device(t, "page_table", dev)
    if t.dim() != 3 or t.dtype is not torch.int32:
        raise ValueError("page_table must be int32 [B, Ht, W]")
    B, Ht, W = t.shape
    sb, sh, sw = t.stride()
    if sw != 1 and W > 1:
        raise ValueError("page_table rows must be contiguous")
    if (batch is not None and B != batch) or (heads is not None and Ht != heads):
        raise ValueError(f"page_table must be [{batch}, {heads if heads is not None else 'Ht'}, W], got {(B, Ht, W)}")
    return t.data_ptr(), sb, sh, Ht, W


@dataclass
class Fp4Pool:
    """K/V pages of one layer on one device in 4-bit floating point.

    ``data`` uint8 [num_pages, page_size / 16, 17 * head_dim] holds 16 rows of K and V, codes and scales, in each
    last dimension.  The byte order there is the kernels' own (``include/intent_attention_b200.h``); ``append_fp4``
    writes it and ``read_fp4`` reads it back.
    """

    num_pages: int
    page_size: int
    head_dim: int
    data: torch.Tensor

    @classmethod
    def allocate(cls, num_pages: int, page_size: int, head_dim: int, device="cuda", zero: bool = False) -> "Fp4Pool":
        """A pool of ``num_pages`` pages (``zero``: all rows 0; otherwise rows hold nothing until written)."""
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if page_size <= 0 or page_size % 16 or page_size > 16384:
            raise ValueError(f"page_size must be a positive multiple of 16 up to 16384, got {page_size}")
        if num_pages < 0:
            raise ValueError("num_pages must not be negative")
        mk = torch.zeros if zero else torch.empty
        return cls(num_pages, page_size, head_dim,
                   mk((num_pages, page_size // 16, 17 * head_dim), dtype=torch.uint8, device=torch.device(device)))

    @property
    def device(self) -> torch.device:
        return self.data.device

    def tensors(self):
        return [self.data]

    def nbytes(self) -> int:
        return self.data.numel()

    def struct(self) -> N.Fp4PoolStruct:
        t = self.data
        if not t.is_cuda:
            _require_cuda(t, "pool data")
        if t.dtype is not torch.uint8 or not t.is_contiguous() \
                or t.numel() != self.num_pages * (self.page_size // 16) * 17 * self.head_dim:
            raise ValueError("pool data must be contiguous uint8 [num_pages, page_size / 16, 17 * head_dim]")
        return N.Fp4PoolStruct(t.data_ptr(), self.num_pages, self.page_size, self.head_dim)


# ---------------------------------------------------------------------- #
#  Rows in and out
# ---------------------------------------------------------------------- #

def _rows_args(dev, k, v, table, positions, counts, dropped=None) -> N.Fp4RowsArgs:
    pt, pt_sb, pt_sh, _, W = table
    B, Ht, n, _ = k.shape
    ksb, ksh, ksn, _ = k.stride()
    vsb, vsh, vsn, _ = v.stride()
    return N.Fp4RowsArgs(k.data_ptr(), v.data_ptr(), _DT[k.dtype], ksb, ksh, ksn, vsb, vsh, vsn, B, Ht, n,
                         pt, pt_sb, pt_sh, W, _index_tensor(positions, "positions", dev, B),
                         _index_tensor(counts, "counts", dev, B), _index_tensor(dropped, "dropped", dev, 1))


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
    two rows of V share their bytes.  After ``grow_sequences`` the counts are
    what the lengths grew by: a slot that was refused may still share its page.
    """
    s, dev = pool.struct(), pool.data.get_device()
    _check_device(k_new, "k_new", dev)
    _check_device(v_new, "v_new", dev)
    shape = k_new.shape
    if len(shape) != 4 or shape != v_new.shape or shape[3] != pool.head_dim:
        raise ValueError(f"k_new / v_new must both be [B, Ht, n, {pool.head_dim}]")
    if k_new.dtype != v_new.dtype or k_new.dtype not in _DT:
        raise ValueError("k_new / v_new must share a float32 / float16 / bfloat16 dtype")
    if k_new.stride(3) != 1:
        k_new = k_new.contiguous()
    if v_new.stride(3) != 1:
        v_new = v_new.contiguous()
    table = _page_table(page_table, dev, shape[0], shape[1])
    a = _rows_args(dev, k_new, v_new, table, positions, counts, dropped)
    with _on(dev):
        N.check(N.lib().iak_fp4_append(ctypes.byref(s), ctypes.byref(a), _raw_stream(dev)), "iak_fp4_append")


def read_fp4(pool: Fp4Pool, page_table: torch.Tensor, positions: Optional[torch.Tensor], num_rows: int,
             counts: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cached tokens ``positions[b] .. positions[b] + num_rows - 1`` as dense (k, v)
    [B, Ht, num_rows, D].  Every value a pool holds is exact in all three float
    types.  Rows from ``counts[b]`` on, and rows of slots or pages that do not
    exist, are 0.  ``out``: a (k, v) pair to write into."""
    s, dev = pool.struct(), pool.data.get_device()
    table = _page_table(page_table, dev)
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    shape = (page_table.shape[0], page_table.shape[1], num_rows, pool.head_dim)
    if out is None:
        if dtype not in _DT:
            raise ValueError("dtype must be float32 / float16 / bfloat16")
        k = torch.empty(shape, dtype=dtype, device=pool.data.device)
        v = torch.empty_like(k)
    else:
        k, v = out
        for name, x in (("out[0]", k), ("out[1]", v)):
            _check_device(x, name, dev)
            if tuple(x.shape) != shape or x.dtype not in _DT or x.dtype != k.dtype:
                raise ValueError(f"{name} must be a {shape} float tensor, both of one dtype")
            if x.stride(3) != 1:
                raise ValueError(f"{name} needs a unit stride along head_dim")
    a = _rows_args(dev, k, v, table, positions, counts)
    with _on(dev):
        N.check(N.lib().iak_fp4_read(ctypes.byref(s), ctypes.byref(a), _raw_stream(dev)), "iak_fp4_read")
    return k, v


# ---------------------------------------------------------------------- #
#  Attention
# ---------------------------------------------------------------------- #

def _decode(q: torch.Tensor, pool: Fp4Pool, page_table: torch.Tensor, lengths: torch.Tensor, sm_scale: float,
            out: Optional[torch.Tensor], out_dtype: Optional[torch.dtype], differential=None) -> torch.Tensor:
    s, dev = pool.struct(), pool.data.get_device()
    _check_device(q, "q", dev)
    shape, strides = q.shape, q.stride()
    dims = len(shape)
    if dims not in (3, 4) or shape[-1] != pool.head_dim:
        raise ValueError(f"q must be [B, Hq, {pool.head_dim}] or [B, Hq, M, {pool.head_dim}], got {tuple(shape)}")
    if q.dtype not in _DT:
        raise ValueError(f"q dtype {q.dtype} unsupported")
    if strides[-1] != 1:
        q = q.contiguous()
        strides = q.stride()
    B, Hq = shape[0], shape[1]
    M = shape[2] if dims == 4 else 1
    if M > N.FP4_MAX_QUERIES:
        raise ValueError(f"at most {N.FP4_MAX_QUERIES} queries per sequence, got {M}: read_fp4 the context for a prompt")
    pt, pt_sb, pt_sh, Ht, W = _page_table(page_table, dev, B)
    if Hq and (Ht == 0 or Hq % Ht):
        raise ValueError(f"query heads ({Hq}) must be a multiple of page-table heads ({Ht})")
    if lengths is None:
        raise ValueError("lengths [B] is required")
    ln = _index_tensor(lengths, "lengths", dev, B)
    if out is not None:
        _check_device(out, "out", dev)
        if out.shape != shape or out.dtype not in _DT or out.stride(-1) != 1:
            raise ValueError(f"out must be a {tuple(shape)} float tensor with a contiguous last dim")
    elif out_dtype is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out_dtype not in _DT:
        raise ValueError(f"out dtype {out_dtype} unsupported")
    else:
        out = torch.empty(shape, dtype=out_dtype, device=q.device)
    os_ = out.stride()
    a = N.Fp4DecodeArgs(q.data_ptr(), _DT[q.dtype], strides[0], strides[1], strides[2] if dims == 4 else 0,
                        out.data_ptr(), _DT[out.dtype], os_[0], os_[1], os_[2] if dims == 4 else 0,
                        B, Hq, Ht, M, pt, pt_sb, pt_sh, W, ln, sm_scale)
    if differential is not None:
        a.differential, a.lam, a.norm_weight, a.eps, a.out_scale = (1, *differential)
    L = N.lib()
    nbytes = ctypes.c_size_t(0)
    ps, pa = ctypes.byref(s), ctypes.byref(a)
    with _on(dev):
        N.check(L.iak_fp4_decode_workspace_size(ps, pa, ctypes.byref(nbytes)), "iak_fp4_decode_workspace_size")
        n = nbytes.value
        # of this call alone: calls on other streams, or captured into other graphs, never share it
        ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
        N.check(L.iak_fp4_decode(ps, pa, ws.data_ptr() if n else None, n, _raw_stream(dev)), "iak_fp4_decode")
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
    ``sm_scale`` defaults to 1 / sqrt(D).  ``out`` may be ``q`` itself.
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
        _check_device(t, name, pool.data.get_device())
        if t.dtype is not torch.float32 or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"{name} must be {n} contiguous float32 values")
        return t.data_ptr()

    if not isinstance(q, torch.Tensor) or q.dim() < 2:
        raise ValueError("q must be [B, Hq, D] or [B, Hq, M, D]")
    lam_ptr = weight(lam, "lam", q.shape[1])
    norm_ptr = None if norm_weight is None else weight(norm_weight, "norm_weight", pool.head_dim)
    scale = 1.0 / math.sqrt(pool.head_dim // 2) if sm_scale is None else float(sm_scale)
    return _decode(q, pool, page_table, lengths, scale, out, out_dtype, (lam_ptr, norm_ptr, float(eps), float(out_scale)))

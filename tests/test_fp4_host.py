"""FP4 cache and page operations without a GPU: the oracle's own definition, the C structs and what the C ABI refuses
before any device call."""

import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from intent_attention import Fp4Pool, SequencePages, append_fp4, compact_pages, paged_decode_fp4
from intent_attention import _native as N
from oracle import fp4 as of

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

STRUCTS = {"iak_fp4_pool": N.Fp4PoolStruct, "iak_fp4_rows_args": N.Fp4RowsArgs, "iak_fp4_decode_args": N.Fp4DecodeArgs,
           "iak_seq_pages": N.SeqPages, "iak_page_planes": N.PagePlanes}


def test_struct_layouts(tmp_path):
    lines = []
    for name, ct in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in ct._fields_]
    src = tmp_path / "t.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "intent_attention_b200.h"\nint main(void) {'
                   + "\n".join(lines) + "return 0; }\n")
    exe = str(tmp_path / "t")
    r = subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", exe], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    for line in subprocess.run([exe], capture_output=True, text=True).stdout.splitlines():
        key, n = line.rsplit(" ", 1)
        name, _, field = key.partition(".")
        ct = STRUCTS[name]
        assert int(n) == (getattr(ct, field).offset if field else ctypes.sizeof(ct)), key


def test_oracle_values():
    x = np.zeros((2, 32))
    x[0, :8] = [6, 5, -5.01, 2.5, 3.5, 0.25, 0.75, 1.25]
    x[1, :3] = [6.5, 1.0, np.nan]
    v = of.values(x)
    assert v[0, :8].tolist() == [6, 4, -6, 2, 4, 0, 1, 1]
    assert v[1, :3].tolist() == [6, 1, 0]            # e = 1: 3.25 -> 3, 0.5 -> 0.5
    # every value is exact in all three float types
    y = of.values(np.random.default_rng(0).standard_normal((100, 64)) * 1000)
    assert (y.astype(np.float16) == y).all()
    assert (torch.from_numpy(y).bfloat16().double().numpy() == y).all()


def _pool():
    p = N.Fp4PoolStruct()
    p.data = 256
    p.num_pages, p.page_size, p.head_dim = 4, 16, 128
    return p


def test_fp4_args_rejected_on_the_host():
    L = N.lib()
    r = ctypes.byref
    for fn, a in ((L.iak_fp4_append, N.Fp4RowsArgs()), (L.iak_fp4_read, N.Fp4RowsArgs())):
        p = _pool()
        assert fn(r(p), r(a), None) == N.IAK_OK                      # nothing to do
        a.batch, a.num_table_heads, a.num_rows, a.table_width = 1, 1, 2, 1
        assert fn(r(p), r(a), None) == N.IAK_ERR_INVALID_ARG         # null rows
        a.dtype = 3
        assert fn(r(p), r(a), None) == N.IAK_ERR_INVALID_ARG
        a.dtype = 0
        for field, value, want in (("head_dim", 96, N.IAK_ERR_UNSUPPORTED), ("page_size", 24, N.IAK_ERR_UNSUPPORTED),
                                   ("page_size", 0, N.IAK_ERR_UNSUPPORTED), ("data", 8, N.IAK_ERR_INVALID_ARG),
                                   ("data", None, N.IAK_ERR_INVALID_ARG), ("num_pages", -1, N.IAK_ERR_INVALID_ARG)):
            p = _pool()
            setattr(p, field, value)
            assert fn(r(p), r(a), None) == want, field
        a.num_rows = -1
        assert fn(r(_pool()), r(a), None) == N.IAK_ERR_INVALID_ARG
    d = N.Fp4DecodeArgs()
    p = _pool()
    call = lambda: L.iak_fp4_decode(r(p), r(d), None, 0, None)       # noqa: E731
    assert call() == N.IAK_OK
    d.batch, d.num_q_heads, d.num_table_heads, d.num_queries, d.table_width = 1, 4, 3, 1, 2
    assert call() == N.IAK_ERR_INVALID_ARG and b"multiple" in L.iak_last_error()
    d.num_table_heads = 2
    assert call() == N.IAK_ERR_INVALID_ARG                           # null q
    d.num_queries = N.FP4_MAX_QUERIES + 1
    assert call() == N.IAK_ERR_UNSUPPORTED
    d.num_queries = 1
    d.q = d.out = d.lengths = d.page_table = 256
    d.sm_scale = float("nan")
    assert call() == N.IAK_ERR_INVALID_ARG
    d.sm_scale, d.differential = 1.0, 1
    assert call() == N.IAK_ERR_INVALID_ARG and b"lam" in L.iak_last_error()
    d.differential, d.table_width = 0, 1 << 30
    assert call() == N.IAK_ERR_UNSUPPORTED
    assert L.iak_fp4_decode_workspace_size(r(p), r(d), None) == N.IAK_ERR_INVALID_ARG


@pytest.mark.parametrize("field,value", [("eps", -1e-6), ("eps", float("nan")), ("eps", 1e39), ("out_scale", 1e39),
                                         ("out_scale", float("nan"))])
def test_differential_numbers_rejected_on_the_host(field, value):
    """What is not finite as a float (1e39 is as a double), and an eps that could make a mean square negative."""
    L = N.lib()
    r = ctypes.byref
    d, p = N.Fp4DecodeArgs(), _pool()
    d.batch, d.num_q_heads, d.num_table_heads, d.num_queries, d.table_width = 1, 4, 2, 1, 2
    d.q = d.out = d.lengths = d.page_table = d.lam = 256
    d.sm_scale, d.out_scale, d.differential = 1.0, 1.0, 1
    setattr(d, field, value)
    n = ctypes.c_size_t(0)
    assert L.iak_fp4_decode_workspace_size(r(p), r(d), r(n)) == N.IAK_ERR_INVALID_ARG and b"eps" in L.iak_last_error()
    assert L.iak_fp4_decode(r(p), r(d), None, 0, None) == N.IAK_ERR_INVALID_ARG


def test_page_args_rejected_on_the_host():
    L = N.lib()
    r = ctypes.byref
    s, pl = N.SeqPages(), N.PagePlanes()
    s.page_size = 16
    n = ctypes.c_size_t(0)
    assert L.iak_pages_grow(r(s), r(pl), None, None, None, 0, None) == N.IAK_OK      # no slots
    s.num_slots, s.num_table_heads, s.table_width, s.num_pages = 2, 1, 4, 8
    assert L.iak_pages_workspace_size(r(s), r(n)) == N.IAK_ERR_INVALID_ARG           # null arrays
    s.refs = s.page_table = s.lengths = 256
    assert L.iak_pages_workspace_size(r(s), r(n)) == N.IAK_OK and n.value >= 4 * 8
    assert L.iak_pages_grow(r(s), r(pl), None, None, None, 0, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_grow(r(s), r(pl), 256, None, 256, 8, None) == N.IAK_ERR_WORKSPACE
    assert L.iak_pages_compact(r(s), r(pl), None, None, 0, None) == N.IAK_ERR_WORKSPACE
    pl.num_planes = 1
    assert L.iak_pages_compact(r(s), r(pl), None, 256, n.value, None) == N.IAK_ERR_INVALID_ARG
    pl.num_planes = 0
    pl.page_tags, pl.tag_bytes = 256, 2
    assert L.iak_pages_compact(r(s), r(pl), None, 256, n.value, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_fork(r(s), 256, 256, -1, None, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_fork(r(s), None, 256, 1, None, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_fork(r(s), 256, 256, 0, None, None) == N.IAK_OK
    assert L.iak_pages_free(r(s), None, 1, None, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_free(r(s), 256, 1 << 30, None, None) == N.IAK_ERR_UNSUPPORTED
    s.page_size = 0
    assert L.iak_pages_free(r(s), 256, 1, None, None) == N.IAK_ERR_INVALID_ARG


def test_shrink_and_wide_tables_rejected_on_the_host():
    L = N.lib()
    r = ctypes.byref
    s, pl = N.SeqPages(), N.PagePlanes()
    s.page_size = 16
    assert L.iak_pages_shrink(None, 256, None, None) == N.IAK_ERR_INVALID_ARG
    assert L.iak_pages_shrink(r(s), None, None, None) == N.IAK_OK                    # no slots
    s.num_slots, s.num_table_heads, s.table_width, s.num_pages = 1024, 2, 1 << 21, 8
    s.refs = s.page_table = s.lengths = 256
    assert L.iak_pages_shrink(r(s), None, None, None) == N.IAK_ERR_INVALID_ARG
    # 1024 rows' pages are counted in 31 bits
    assert L.iak_pages_grow(r(s), r(pl), 256, None, 256, 1 << 30, None) == N.IAK_ERR_UNSUPPORTED
    pl.num_planes, pl.base[0], pl.bytes[0] = 1, 256, 1 << 50
    assert L.iak_pages_grow(r(s), r(pl), 256, None, 256, 1 << 30, None) == N.IAK_ERR_UNSUPPORTED


def test_imports_on_a_torch_build_without_cuda():
    """The package's host side (router, policies, layouts) needs none of torch's CUDA entry points."""
    code = """
import torch
for name in [n for n in vars(torch._C) if n.startswith("_cuda_")]:
    delattr(torch._C, name)
import intent_attention as ia
assert ia.Fp4Pool.allocate(2, 16, 64, device="cpu").nbytes() == 2 * 17 * 64
assert ia.SequencePages.allocate(2, 16, 1, 1, 2, device="cpu").lengths.tolist() == [0]
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.join(ROOT, "intent-attention-kernel_b200"),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_go_to_the_tensors_device(monkeypatch):
    """Another device than the current one is made current for the call, and its own stream taken."""
    from intent_attention import fp4_cache as fc
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 1000 + dev, raising=False)
    assert fc._on(0) is fc._NO_SWITCH
    other = fc._on(1)
    assert isinstance(other, torch.cuda.device) and other.idx == 1
    assert fc._raw_stream(1) == 1001


def test_no_cpu_fallback():
    for args in ((4, 16, 96), (4, 24, 128), (-1, 16, 128)):
        with pytest.raises(ValueError):
            Fp4Pool.allocate(*args, device="cpu")
    pool = Fp4Pool.allocate(4, 16, 128, device="cpu")
    assert pool.nbytes() == 4 * 16 * 2 * (64 + 4)
    k = torch.zeros(1, 1, 2, 128)
    table, n = torch.zeros(1, 1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for f in (lambda: append_fp4(pool, k, k, table), lambda: paged_decode_fp4(k[:, :, 0], pool, table, n),
              lambda: compact_pages(pool, SequencePages.allocate(4, 16, 1, 1, 2, device="cpu"))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()

"""Paged-cache checks that need no GPU: struct layouts, argument errors of the C
ABI before any launch, and the refusals of the Python ops."""

import ctypes
import math
import os
import re
import subprocess
import sys

import pytest
import torch

import ssa_b200 as ssa
from ssa_b200 import _lib as L
from ssa_b200.build import build
from test_abi import _c_layout


@pytest.fixture(scope="module")
def lib():
    build()
    return L.lib()


@pytest.mark.parametrize("cls,name", [(L.SsaPagedCache, "SsaPagedCache"), (L.SsaPagedAppendArgs, "SsaPagedAppendArgs"),
                                      (L.SsaPagedAttnArgs, "SsaPagedAttnArgs"),
                                      (L.SsaPagedEvictArgs, "SsaPagedEvictArgs")])
def test_ctypes_structs_match_c_layout(cls, name):
    fields = [f for f, _ in cls._fields_]
    size, offsets = _c_layout(name, fields)
    assert ctypes.sizeof(cls) == size
    assert [getattr(cls, f).offset for f in fields] == offsets


def _fill(cls, vals, over):
    a = cls()
    for k, v in {**vals, **over}.items():
        setattr(a, k, v)
    return a


def _cache(**over):
    return _fill(L.SsaPagedCache, dict(
        batch=2, max_pages=4, page_size=16, h_kv=2, d=64, dtype=L.SSA_BF16, num_pages=8,
        k_pages=0x1000, k_stride_p=2048, k_stride_n=128, k_stride_h=64,
        v_pages=0x2000, v_stride_p=2048, v_stride_n=128, v_stride_h=64,
        page_table=0x3000, table_stride=4, kv_lens=0x4000), over)


def _attn(**over):
    return _fill(L.SsaPagedAttnArgs, dict(
        rows=3, q_starts=0x5000, h_q=8, causal=1, scale=8.0, q=0x6000, q_stride_n=512, q_stride_h=64,
        out=0x7000, out_stride_n=512, out_stride_h=64), over)


CACHE_ERRORS = [
    (dict(batch=-1), 1), (dict(max_pages=-1), 1), (dict(num_pages=-1), 1), (dict(batch=70000), 2),
    (dict(page_size=0), 2), (dict(page_size=1025), 2), (dict(h_kv=0), 1), (dict(d=4), 2), (dict(d=264), 2),
    (dict(d=60), 2), (dict(dtype=7), 1), (dict(max_pages=1 << 27), 2), (dict(kv_lens=None), 1),
    (dict(page_table=None), 1), (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(k_pages=0x1008), 4),
    (dict(v_stride_n=132), 4), (dict(k_stride_p=2052), 4),
]


@pytest.mark.parametrize("over,code", CACHE_ERRORS)
def test_cache_argument_errors(lib, over, code):
    c, a = _cache(**over), _attn()
    assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), None, 0, None) == code, lib.ssa_last_error()
    assert lib.ssa_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(a)) == 0
    p = _fill(L.SsaPagedAppendArgs, dict(rows=1, q_starts=0x5000, k_new=0x6000, v_new=0x6000), {})
    assert lib.ssa_paged_append(ctypes.byref(c), ctypes.byref(p), None) == code
    e = _fill(L.SsaPagedEvictArgs, dict(budget=4), {})
    assert lib.ssa_paged_evict(ctypes.byref(c), ctypes.byref(e), None) == code


@pytest.mark.parametrize("over,code", [
    (dict(rows=-1), 1), (dict(rows=1 << 31), 1), (dict(q_starts=None), 1), (dict(h_q=7), 1), (dict(h_q=0), 1),
    (dict(h_q=34), 2), (dict(scale=0.0), 1), (dict(scale=math.inf), 1), (dict(scale=math.nan), 1), (dict(scale=1e-45), 1),
    (dict(q=None), 1), (dict(out=None), 1), (dict(q=0x6004), 4), (dict(out_stride_h=68), 4),
])
def test_attention_argument_errors(lib, over, code):
    c, a = _cache(), _attn(**over)
    assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), None, 0, None) == code, lib.ssa_last_error()


def test_attention_needs_its_workspace(lib):
    c, a = _cache(), _attn()
    need = lib.ssa_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(a))
    assert need > 0
    assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 3
    assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), 0x10000, need - 1, None) == 3
    assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), 0x10008, need, None) == 4
    assert lib.ssa_paged_attn(ctypes.byref(c), None, None, 0, None) == 1
    assert lib.ssa_paged_attn(None, ctypes.byref(a), None, 0, None) == 1


@pytest.mark.parametrize("over,code", [
    (dict(budget=0), 1), (dict(recent=-1), 1), (dict(recent=5), 1), (dict(new_max_pages=-1), 1),
    (dict(kept=None), 1), (dict(new_lens=None), 1), (dict(new_table=None), 1),
])
def test_evict_argument_errors(lib, over, code):
    c = _cache(weights=0x8000)
    e = _fill(L.SsaPagedEvictArgs, dict(budget=4, recent=1, new_max_pages=1, new_table=0x9000, new_table_stride=1,
                                        kept=0xa000, new_lens=0xb000), over)
    assert lib.ssa_paged_evict(ctypes.byref(c), ctypes.byref(e), None) == code, lib.ssa_last_error()


def test_evict_needs_weights_and_append_its_rows(lib):
    c = _cache()
    e = _fill(L.SsaPagedEvictArgs, dict(budget=4), {})
    assert lib.ssa_paged_evict(ctypes.byref(c), ctypes.byref(e), None) == 1
    for over, code in ((dict(k_new=None), 1), (dict(v_new=0x6008), 4), (dict(rows=-1), 1), (dict(q_starts=None), 1)):
        p = _fill(L.SsaPagedAppendArgs, dict(rows=1, q_starts=0x5000, k_new=0x6000, v_new=0x6000), over)
        assert lib.ssa_paged_append(ctypes.byref(c), ctypes.byref(p), None) == code


def test_cpu_tensors_raise_no_fallback():
    k = torch.zeros(4, 16, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ssa.paged_attention(torch.zeros(1, 4, 64), k, k, i[None, :1], i, i[:1]),
                 lambda: ssa.paged_append(k[0, :1], k[0, :1], k, k, i[None, :1], i, i[:1]),
                 lambda: ssa.paged_evict(k, k, k[..., 0], i[None, :1], i[:1], i[None, :1], 4)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_workspace_of_a_call_without_work(lib):
    """No sequence or no row: a size all the same, and a call that does nothing.
    In a process of its own: a fault there would take this one along."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = f"""
import ctypes, sys
sys.path[:0] = [{root!r}, {os.path.join(root, 'tests')!r}]
from test_paged_cpu import L, _attn, _cache
lib = L.lib()
for dtype in (L.SSA_F32, L.SSA_BF16, L.SSA_F16):
    for batch, rows in ((0, 0), (0, 5), (2, 0)):
        c, a = _cache(batch=batch, dtype=dtype), _attn(rows=rows)
        need = lib.ssa_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(a))
        assert need == L.SSA_PAGED_ZEROED, (dtype, batch, rows, need)
        assert lib.ssa_paged_attn(ctypes.byref(c), ctypes.byref(a), None, 0, None) == 0
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr)


@pytest.mark.parametrize("dtype,d", [(L.SSA_BF16, 128), (L.SSA_F16, 64), (L.SSA_F32, 64), (L.SSA_BF16, 96)])
def test_workspace_of_weights_with_wide_tables(lib, dtype, d):
    """The kept scores of single tokens follow the table's width: they are bounded."""
    c = _cache(batch=4096, max_pages=2048, page_size=64, h_kv=8, d=d, dtype=dtype, weights=0x8000,
               num_pages=8, k_stride_p=64 * 8 * d, k_stride_n=8 * d, k_stride_h=d, v_stride_p=64 * 8 * d,
               v_stride_n=8 * d, v_stride_h=d, table_stride=2048)
    a = _attn(rows=4096, h_q=32, q_stride_n=32 * d, q_stride_h=d, out_stride_n=32 * d, out_stride_h=d)
    assert 0 < lib.ssa_paged_attn_workspace_size(ctypes.byref(c), ctypes.byref(a)) < 4.1 * 2 ** 30, lib.ssa_last_error()


def test_dependent_kernels_do_not_read_results_through_the_read_only_cache():
    """They start while the kernel before them writes, and __ldg is for what nothing writes
    while the reader runs."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ssa_b200", "csrc")
    for name in sorted(os.listdir(csrc)):
        if name.startswith("paged"):
            with open(os.path.join(csrc, name)) as f:
                found = re.findall(r"__ldg\(\s*(?:\w+\.)*(?:lse2|lse|part|split|scores|kept)\b", f.read())
            assert not found, (name, found)

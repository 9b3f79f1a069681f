"""Refusals and plans of the cache, shared-prefix and rotary entry points, without a GPU: nothing is launched."""

import ctypes as C
import os
import subprocess
import tempfile

import pytest
import torch

from torch_neuronx_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rotary(**change):
    p = _lib.RotaryParams()
    p.struct_size = C.sizeof(p)
    p.dtype, p.device = _lib.BF16, 0
    p.x[0] = p.x[1] = p.y[0] = p.y[1] = 4096
    p.heads[0], p.heads[1] = 4, 2
    p.B, p.L, p.D, p.rot, p.axes = 2, 8, 64, 64, 2
    p.section[:2] = [12, 20]
    p.positions = p.inv_freq = 4096
    for name, value in change.items():
        setattr(p, name, value)
    return p


def _rows(**change):
    p = _lib.CacheRowsParams()
    p.struct_size = C.sizeof(p)
    p.dtype, p.device, p.page_size = _lib.F16, 0, 16
    for name in ("k", "v", "k_pages", "v_pages", "k_scales", "v_scales", "block_table", "start", "lens"):
        setattr(p, name, 4096)
    p.k_pages_stride[:] = p.v_pages_stride[:] = [1024, 64, 64]
    p.B, p.Hkv, p.L, p.D, p.block_table_stride, p.n_pages = 2, 1, 5, 64, 3, 4
    for name, value in change.items():
        setattr(p, name, value)
    return p


def _decode(**change):
    p = _lib.CacheDecodeParams()
    p.struct_size = C.sizeof(p)
    p.dtype, p.device, p.page_size = _lib.BF16, 0, 16
    for name in ("q", "out", "k_pages", "v_pages", "k_scales", "v_scales", "block_table", "kv_lens", "prefix_table"):
        setattr(p, name, 4096)
    p.q_stride[:] = p.out_stride[:] = [1024, 128, 1]
    p.k_pages_stride[:] = p.v_pages_stride[:] = [4096, 128, 256]
    p.B, p.Hq, p.Hkv, p.D, p.scale = 4, 8, 2, 128, 0.1
    p.n_pages, p.block_table_stride, p.prefix_len = 100, 10, 0
    for name, value in change.items():
        setattr(p, name, value)
    return p


def _triple(*v):
    return (C.c_int64 * 3)(*v)


@pytest.mark.parametrize("change,code", [
    ({"struct_size": 4}, _lib.ERR_STRUCT), ({"dtype": 7}, _lib.ERR_DTYPE), ({"rot": 63}, _lib.ERR_SHAPE), ({"rot": 66}, _lib.ERR_SHAPE),
    ({"axes": 5}, _lib.ERR_SHAPE), ({"axes": 1}, _lib.ERR_SHAPE), ({"B": 0}, _lib.ERR_SHAPE), ({"positions": None}, _lib.ERR_NULL),
    ({"B": 70000}, _lib.ERR_UNSUPPORTED),
])
def test_rotary_refusals(change, code):
    assert _lib.load().b200_sdpa_rotary(C.byref(_rotary(**change)), None) == code


@pytest.mark.parametrize("change,code", [
    ({"struct_size": 4}, _lib.ERR_STRUCT), ({"dtype": _lib.F32}, _lib.ERR_DTYPE), ({"page_size": 12}, _lib.ERR_SHAPE), ({"L": 0}, _lib.ERR_SHAPE),
    ({"D": 24}, _lib.ERR_UNSUPPORTED), ({"D": 272}, _lib.ERR_UNSUPPORTED), ({"n_pages": 0}, _lib.ERR_SHAPE), ({"k_scales": None}, _lib.ERR_NULL),
    ({"block_table": None}, _lib.ERR_NULL), ({"k_pages": 4104}, _lib.ERR_ALIGNMENT), ({"v_pages_stride": _triple(1024, 72, 64)}, _lib.ERR_ALIGNMENT),
    ({"block_table_stride": 1 << 28}, _lib.ERR_UNSUPPORTED),
])
def test_rows_refusals(change, code):
    lib = _lib.load()
    assert lib.b200_sdpa_cache_write(C.byref(_rows(**change)), None) == code
    assert lib.b200_sdpa_cache_read(C.byref(_rows(**change)), None) == code


def test_rows_need_their_vectors():
    lib = _lib.load()
    assert lib.b200_sdpa_cache_write(C.byref(_rows(start=None)), None) == _lib.ERR_NULL
    assert lib.b200_sdpa_cache_read(C.byref(_rows(lens=None)), None) == _lib.ERR_NULL
    assert lib.b200_sdpa_cache_write(None, None) == lib.b200_sdpa_rotary(None, None) == _lib.ERR_NULL


def _plan(p):
    plan = _lib.Plan()
    plan.struct_size = C.sizeof(plan)
    return _lib.load().b200_sdpa_cache_decode_plan(C.byref(p), C.byref(plan)), plan


@pytest.mark.parametrize("change,code", [
    ({"struct_size": 4}, _lib.ERR_STRUCT), ({"dtype": _lib.F32}, _lib.ERR_DTYPE), ({"Hq": 7}, _lib.ERR_SHAPE), ({"D": 96}, _lib.ERR_UNSUPPORTED),
    ({"scale": -1.0}, _lib.ERR_UNSUPPORTED), ({"scale": float("nan")}, _lib.ERR_UNSUPPORTED), ({"page_size": 0}, _lib.ERR_SHAPE),
    ({"prefix_len": -1}, _lib.ERR_SHAPE), ({"prefix_len": 5, "prefix_table": None}, _lib.ERR_NULL), ({"v_scales": None}, _lib.ERR_NULL),
    ({"k_scales": None, "v_scales": None}, _lib.ERR_UNSUPPORTED), ({"kv_lens": None}, _lib.ERR_NULL), ({"k_pages": 4097}, _lib.ERR_ALIGNMENT),
    ({"block_table_stride": 1 << 27}, _lib.ERR_UNSUPPORTED), ({"prefix_len": 0x7FFFFFFF}, _lib.ERR_UNSUPPORTED),
    ({"k_scales_stride": _triple(1 << 32, 1, 1)}, _lib.ERR_UNSUPPORTED), ({"prefix_len": 5, "q": 4098}, _lib.ERR_ALIGNMENT), ({"prefix_len": 5, "Hq": 258}, _lib.ERR_UNSUPPORTED), ({"B": 70000}, _lib.ERR_UNSUPPORTED),
])
def test_decode_refusals(change, code):
    assert _plan(_decode(**change))[0] == code
    assert _lib.load().b200_sdpa_cache_decode(C.byref(_decode(**change)), None) == code


def test_decode_plans():
    rc, plan = _plan(_decode())
    assert rc == _lib.OK and plan.launches == 2 and plan.kv_splits >= 1
    assert plan.workspace_bytes >= 8 * plan.kv_splits * 130 * 4
    # a range longer than any table is the whole table
    for scales in ({}, {"k_scales": None, "v_scales": None, "prefix_len": 100}):
        rc, whole = _plan(_decode(kv_chunk=0x7FFFFFFF, **scales))
        assert rc == _lib.OK and whole.kv_splits >= 1 and whole.workspace_bytes < 1 << 32
    # few sequences: the prefix is an entry before each one's own keys, in the same two launches; many: gathered, multiplied once
    rc, shared = _plan(_decode(prefix_len=1000))
    assert rc == _lib.OK and shared.launches == 2 and shared.workspace_bytes > plan.workspace_bytes
    rc, shared = _plan(_decode(prefix_len=4000, B=128))
    assert rc == _lib.OK and shared.launches == 4 and shared.workspace_bytes > 2 * 4000 * 2 * 128 * 2
    rc, only = _plan(_decode(prefix_len=4000, B=128, block_table_stride=0, block_table=None))
    assert rc == _lib.OK and only.kv_splits == 0 and only.launches == 3
    # a 16-bit prefix likewise, or it is read in its pages, or gathered from pages of fewer than 8 rows
    for more, launches in (({}, 2), ({"B": 500}, 3), ({"B": 500, "page_size": 4}, 4)):
        rc, sixteen = _plan(_decode(prefix_len=1000, k_scales=None, v_scales=None, **more))
        assert rc == _lib.OK and sixteen.launches == launches


def test_struct_layout_matches_the_header():
    code = r"""
#include <stdio.h>
#include "b200_sdpa.h"
int main(void) {
  printf("%zu %zu %zu\n", sizeof(B200RotaryParams), offsetof(B200RotaryParams, section), offsetof(B200RotaryParams, inv_freq));
  printf("%zu %zu %zu\n", sizeof(B200CacheRowsParams), offsetof(B200CacheRowsParams, B), offsetof(B200CacheRowsParams, start));
  printf("%zu %zu %zu\n", sizeof(B200CacheDecodeParams), offsetof(B200CacheDecodeParams, scale), offsetof(B200CacheDecodeParams, workspace));
  return 0;
}
"""
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "s.c"), os.path.join(d, "s")
        with open(src, "w") as f:
            f.write(code)
        subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), src, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    R, W, D = _lib.RotaryParams, _lib.CacheRowsParams, _lib.CacheDecodeParams
    assert got == [C.sizeof(R), R.section.offset, R.inv_freq.offset, C.sizeof(W), W.B.offset, W.start.offset,
                   C.sizeof(D), D.scale.offset, D.workspace.offset]


def test_tensors_of_the_host_are_refused():
    import torch_neuronx_b200 as T

    q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
    kp = torch.zeros(2, 16, 1, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    ks = torch.zeros(2, 16, 1, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        T.rotary_embedding(q, None, lens.view(1, 1), torch.ones(32))
    with pytest.raises(ValueError, match="CUDA"):
        T.paged_write(q[:, :1], q[:, :1], kp, kp, ks, ks, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        T.paged_read(kp, kp, ks, ks, table, lens)
    with pytest.raises(ValueError, match="CUDA"):
        T.paged_decode(q, kp, kp, table, lens, k_scales=ks, v_scales=ks)
    with pytest.raises(ValueError, match="CUDA"):
        T.shared_prefix_decode(q, kp, kp, table[0], 4, table, lens, k_scales=ks, v_scales=ks)

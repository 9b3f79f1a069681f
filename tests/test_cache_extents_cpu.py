"""Extents near and beyond 2^31 are refused before anything is launched."""

import ctypes as C

import pytest

from tests.test_cache_abi_cpu import _rotary, _rows
from torch_neuronx_b200 import _lib


@pytest.mark.parametrize("n", [0x7FFFFFFF, 0x7FFFFFF0])
def test_row_counts_near_2_31(n):
    lib = _lib.load()
    assert lib.b200_sdpa_rotary(C.byref(_rotary(L=n)), None) == _lib.ERR_UNSUPPORTED
    assert lib.b200_sdpa_cache_write(C.byref(_rows(L=n)), None) == _lib.ERR_UNSUPPORTED
    assert lib.b200_sdpa_cache_read(C.byref(_rows(L=n)), None) == _lib.ERR_UNSUPPORTED

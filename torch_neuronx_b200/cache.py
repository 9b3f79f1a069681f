"""The 8-bit paged key/value cache, and decode for a batch that shares a prefix.

An 8-bit cache is two pools of e4m3 values beside two of row scales: ``(pages, page_size, Hkv, D)`` of
``torch.float8_e4m3fn`` and ``(pages, page_size, Hkv)`` of ``torch.float8_e8m0fnu`` for ``layout="NHD"``,
``(pages, Hkv, page_size, D)`` and ``(pages, Hkv, page_size)`` for ``"HND"``.  A row (one token, one head) stands for
``value * scale``; the scale is the least power of two with which the row fits e4m3.  Pages, block tables and lengths are
those of :func:`ops.paged_decode`.  No gradient flows through any of this, and a trace cannot record it.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib, ops

_HALF = (torch.float16, torch.bfloat16)
_SCALE_DTYPES = (torch.float8_e8m0fnu, torch.uint8)


_LAYOUTS = {"NHD": 1, "HND": 2}


def _native():
    """The direct entry points, where nothing is tracing."""
    return None if _lib.native is None or torch.compiler.is_compiling() else _lib.native


def _dims(layout: str):
    """(head dimension, row dimension) of a pool."""
    if layout not in ("NHD", "HND"):
        raise ValueError("layout must be 'NHD' or 'HND'")
    return (2, 1) if layout == "NHD" else (1, 2)


def _check_pools(op, k_pages, v_pages, k_scales, v_scales, device, quantised=True):
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape:
        raise RuntimeError(f"{op}: k_pages and v_pages must be 4-D page pools of the same shape")
    if k_pages.shape[0] == 0:
        raise RuntimeError(f"{op}: the page pools are empty")
    if k_pages.device != device or v_pages.device != device or device.type != "cuda":
        raise ValueError(f"Expected CUDA tensors on one device, got {device}, {k_pages.device}, {v_pages.device}")
    if k_pages.stride(3) != 1 or v_pages.stride(3) != 1:
        raise RuntimeError(f"{op}: the page pools must have a unit inner stride")
    if not quantised:
        return
    if k_pages.dtype != torch.float8_e4m3fn or v_pages.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"{op}: the pools of an 8-bit cache must be float8_e4m3fn")
    for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
        if t is None or t.dtype not in _SCALE_DTYPES or t.shape != k_pages.shape[:3] or t.device != device:
            raise RuntimeError(f"{op}: {name} must be a float8_e8m0fnu tensor of the pools' first three extents on their device")


def _check_vector(op, name, t, B, device):
    if t.dtype != torch.int32 or t.shape != (B,) or t.device != device:
        raise RuntimeError(f"{op}: {name} must be an int32 CUDA tensor of shape (B,) on the pools' device")
    return t.contiguous()


def _check_table(op, block_table, B, device):
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or block_table.device != device:
        raise RuntimeError(f"{op}: block_table must be an int32 CUDA tensor of shape (B, max_pages)")
    return block_table.contiguous()


def _order(t, hd, rd):
    return [t.stride(0), t.stride(hd), t.stride(rd)]


def _rows_params(op, key, value, k_pages, v_pages, k_scales, v_scales, block_table, layout):
    hd, rd = _dims(layout)
    _check_pools(op, k_pages, v_pages, k_scales, v_scales, key.device)
    B, Hkv, L, D = key.shape
    if (k_pages.shape[hd], k_pages.shape[3]) != (Hkv, D):
        raise RuntimeError(f"{op}: the pools hold rows of {k_pages.shape[hd]} heads x {k_pages.shape[3]}, not {Hkv} x {D}")
    p = _lib.CacheRowsParams()
    p.struct_size = C.sizeof(_lib.CacheRowsParams)
    p.dtype = ops._DTYPE_CODE[key.dtype]
    p.device = ops._device_index(key)
    p.page_size = k_pages.shape[rd]
    p.k, p.v = key.data_ptr(), value.data_ptr()
    p.k_stride[:] = key.stride()[:3]
    p.v_stride[:] = value.stride()[:3]
    p.k_pages, p.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
    p.k_pages_stride[:] = _order(k_pages, hd, rd)
    p.v_pages_stride[:] = _order(v_pages, hd, rd)
    p.k_scales, p.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
    p.k_scales_stride[:] = _order(k_scales, hd, rd)
    p.v_scales_stride[:] = _order(v_scales, hd, rd)
    p.B, p.Hkv, p.L, p.D = B, Hkv, L, D
    p.block_table = block_table.data_ptr()
    p.block_table_stride = block_table.shape[1]
    p.n_pages = k_pages.shape[0]
    p.status = ops._status_word(p.device).data_ptr()
    return p


def _launch(name, p):
    rc = getattr(_lib.load(), name)(C.byref(p), C.c_void_p(torch.cuda.current_stream(p.device).cuda_stream))
    if rc != _lib.OK:
        raise RuntimeError(f"{name}: {_lib.strerror(rc)}")


def paged_write(
    key: torch.Tensor,
    value: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    start: torch.Tensor,
    *,
    lens: Optional[torch.Tensor] = None,
    layout: str = "NHD",
) -> None:
    """Quantise key and value rows into an 8-bit paged cache, in place.

    ``key`` and ``value`` are ``(B, Hkv, L, D)`` in fp16 or bf16, any strides with a unit inner stride, ``D`` a multiple
    of 16 up to 256; row ``i`` of sequence ``b`` becomes position ``start[b] + i`` for ``i < lens[b]`` (``i < L`` without ``lens``; rows
    of padding are not read into the cache).  A row's scale is the least power of two, from ``2^-127`` on, with which its largest magnitude is at most 448 (1
    for a row of zeros); its values are rounded once, to e4m3.  A row with a NaN or an infinity reads back as NaN.  A position
    behind the table's last page, or a page number outside the pool, drops the row and is reported by
    :func:`ops.check_device_status`.  Two rows of one call must not have the same place."""
    native = _native()
    if native is not None and layout in _LAYOUTS and native.paged_write(
            key, value, k_pages, v_pages, k_scales, v_scales, block_table, start, lens, _LAYOUTS[layout]):
        return
    ops._check_visible("paged_write", key, value)
    if key.dim() != 4 or value.shape != key.shape:
        raise RuntimeError("paged_write: key and value must be 4-D (B, Hkv, L, D) and of the same shape")
    if key.dtype not in _HALF or value.dtype != key.dtype or value.device != key.device:
        raise RuntimeError("paged_write: key and value must share a float16 or bfloat16 dtype and a device")
    if key.shape[3] % 16 or not 16 <= key.shape[3] <= 256 or (key.numel() and (key.stride(3) != 1 or value.stride(3) != 1)):
        raise RuntimeError("paged_write: the head dim must be a multiple of 16 up to 256 with a unit inner stride")
    if max(key.shape) > ops._MOST:
        raise RuntimeError("paged_write: extents are counted in 32 bits")
    B = key.shape[0]
    block_table = _check_table("paged_write", block_table, B, key.device)
    start = _check_vector("paged_write", "start", start, B, key.device)
    if lens is not None:
        lens = _check_vector("paged_write", "lens", lens, B, key.device)
    p = _rows_params("paged_write", key, value, k_pages, v_pages, k_scales, v_scales, block_table, layout)
    if key.numel() == 0:
        return
    p.start = start.data_ptr()
    if lens is not None:
        p.lens = lens.data_ptr()
    _launch("b200_sdpa_cache_write", p)


def paged_read(
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    k_scales: torch.Tensor,
    v_scales: torch.Tensor,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    *,
    max_len: Optional[int] = None,
    dtype: torch.dtype = torch.bfloat16,
    layout: str = "NHD",
    out: Optional[tuple] = None,
):
    """The first ``max_len`` cached rows of each sequence as dense ``(B, Hkv, max_len, D)`` keys and values in fp16 or
    bf16 -- what :func:`ops.sdpa_forward` takes for the next chunk of a prompt.  Rows at or behind ``kv_lens[b]`` are zeros.
    ``max_len`` is the table's capacity by default.  bf16 holds every cached value exactly but ``2^128``, to which the write rounds
    bf16 magnitudes from ``248 * 2^120`` on and which is an infinity there; fp16 rounds those below ``2^-14`` and overflows beyond 65504.  ``out`` is a pair of tensors to write into (any strides with a unit inner stride)."""
    native = _native()
    if native is not None and layout in _LAYOUTS and out is None and dtype in _HALF:
        got = native.paged_read(k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, max_len, dtype == torch.bfloat16, _LAYOUTS[layout])
        if got is not None:
            return got
    ops._check_visible("paged_read", k_pages, v_pages)
    hd, rd = _dims(layout)
    if dtype not in _HALF:
        raise RuntimeError("paged_read: dtype must be float16 or bfloat16")
    _check_pools("paged_read", k_pages, v_pages, k_scales, v_scales, k_pages.device)
    if block_table.dim() != 2:
        raise RuntimeError("paged_read: block_table must be an int32 CUDA tensor of shape (B, max_pages)")
    B, Hkv, D = block_table.shape[0], k_pages.shape[hd], k_pages.shape[3]
    block_table = _check_table("paged_read", block_table, B, k_pages.device)
    kv_lens = _check_vector("paged_read", "kv_lens", kv_lens, B, k_pages.device)
    if D % 16 or not 16 <= D <= 256:
        raise RuntimeError("paged_read: the head dim must be a multiple of 16 up to 256")
    capacity = block_table.shape[1] * k_pages.shape[rd]
    L = capacity if max_len is None else int(max_len)
    if not 0 <= L <= capacity:
        raise RuntimeError(f"paged_read: max_len {L} is not within the table's capacity of {capacity} rows")
    if out is None:
        key, value = (torch.empty((B, Hkv, L, D), dtype=dtype, device=k_pages.device) for _ in range(2))
    else:
        key, value = out
        for t in (key, value):
            if t.shape != (B, Hkv, L, D) or t.dtype != dtype or t.device != k_pages.device or (t.numel() and t.stride(3) != 1):
                raise RuntimeError("paged_read: out must be two (B, Hkv, max_len, D) tensors of dtype with unit inner stride")
    if key.numel() == 0:
        return key, value
    p = _rows_params("paged_read", key, value, k_pages, v_pages, k_scales, v_scales, block_table, layout)
    p.lens = kv_lens.data_ptr()
    _launch("b200_sdpa_cache_read", p)
    return key, value


def shared_prefix_decode(
    query: torch.Tensor,
    k_pages: torch.Tensor,
    v_pages: torch.Tensor,
    prefix_table: torch.Tensor,
    prefix_len: int,
    block_table: torch.Tensor,
    kv_lens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    layout: str = "NHD",
    out: Optional[torch.Tensor] = None,
    lse: Optional[torch.Tensor] = None,
    need_lse: bool = False,
    kv_chunk: int = 0,
    k_scales: Optional[torch.Tensor] = None,
    v_scales: Optional[torch.Tensor] = None,
):
    """One decode step of a batch whose sequences all start with the same cached prefix; returns ``(out, lse)``.

    Sequence ``b`` attends to the ``prefix_len`` keys in the pages of ``prefix_table`` (int32, ``(pages,)``) and then to its own
    ``kv_lens[b]`` keys (0 is allowed) in the pages of ``block_table[b]`` -- which does not list the prefix's pages.  The result is
    that of :func:`ops.paged_decode` over the joined tables, but the prefix is read and multiplied once for the whole batch (a
    short prefix of few sequences is read for each of them, where that is faster), and sums are taken in another order.  As there,
    probabilities are rounded to the type of a 16-bit cache before they meet the values, and carried as two 16-bit parts for an 8-bit one.
    ``query`` is ``(B, Hq, 1, D)`` with D 64 or 128 and at most 128 query heads for a key head; the pools are in its dtype, or 8-bit with
    ``k_scales`` and ``v_scales`` (cached values of an 8-bit prefix beyond the query type's largest number, 65504 or
    ``255 * 2^120``, may count as that).  ``prefix_len`` is a number of the host, part of a captured graph."""
    if int(prefix_len) < 0:
        raise RuntimeError("shared_prefix_decode: prefix_len must not be negative")
    if prefix_table.dtype != torch.int32 or prefix_table.dim() != 1 or prefix_table.device != query.device:
        raise RuntimeError("shared_prefix_decode: prefix_table must be an int32 CUDA tensor of shape (pages,)")
    return _decode("shared_prefix_decode", query, k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, scale, layout, out, lse,
                   need_lse, kv_chunk, prefix_table.contiguous(), int(prefix_len))


def decode_8bit(query, k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, *, scale, layout, out, lse, need_lse, kv_chunk):
    """:func:`ops.paged_decode` against an 8-bit cache."""
    if k_scales is None or v_scales is None:
        raise RuntimeError("paged_decode: k_scales and v_scales go together")
    return _decode("paged_decode", query, k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, scale, layout, out, lse,
                   need_lse, kv_chunk, None, 0)


def _decode(op, query, k_pages, v_pages, k_scales, v_scales, block_table, kv_lens, scale, layout, out, lse, need_lse, kv_chunk,
            prefix_table, prefix_len):
    native = _native()
    if native is not None and layout in _LAYOUTS:
        got = native.cache_decode(query, k_pages, v_pages, k_scales, v_scales, prefix_table, prefix_len, block_table, kv_lens, scale,
                                  _LAYOUTS[layout], out, lse, need_lse, kv_chunk)
        if got is not None:
            return got
    ops._check_visible(op, query, k_pages, v_pages)
    hd, rd = _dims(layout)
    if query.dim() != 4 or query.shape[2] != 1:
        raise RuntimeError(f"{op}: query must be (B, Hq, 1, D) and the page pools 4-D")
    quantised = k_scales is not None or v_scales is not None
    if query.dtype not in _HALF or (not quantised and (k_pages.dtype != query.dtype or v_pages.dtype != query.dtype)):
        raise RuntimeError(f"{op}: query must be float16 or bfloat16, and the page pools of its dtype or 8-bit with scales")
    _check_pools(op, k_pages, v_pages, k_scales, v_scales, query.device, quantised)
    B, Hq, _, D = query.shape
    Hkv, page_size = k_pages.shape[hd], k_pages.shape[rd]
    if k_pages.shape[3] != D or D not in (64, 128):
        raise RuntimeError(f"{op}: the pools must have the query's head dim, 64 or 128")
    if Hkv == 0 or Hq % Hkv != 0:
        raise RuntimeError("SDPA: Number of heads in key and value must divide the number of heads in query")
    block_table = _check_table(op, block_table, B, query.device)
    kv_lens = _check_vector(op, "kv_lens", kv_lens, B, query.device)
    if prefix_len > 0 and prefix_table.shape[0] * page_size < prefix_len:
        raise RuntimeError(f"{op}: prefix_table has room for {prefix_table.shape[0] * page_size} keys, prefix_len is {prefix_len}")
    if out is None:
        out = torch.empty_like(query)
    elif out.shape != query.shape or out.dtype != query.dtype or out.device != query.device:
        raise RuntimeError(f"{op}: out must match the query in shape, dtype and device")
    if lse is None:
        lse = torch.empty((B, Hq, 1), dtype=torch.float32, device=query.device) if need_lse else None
    elif tuple(lse.shape) != (B, Hq, 1) or lse.dtype != torch.float32 or lse.device != query.device:
        raise RuntimeError(f"{op}: lse must be an fp32 tensor of shape (B, Hq, 1) on the query's device")
    if query.numel() == 0:
        return out, lse
    if prefix_len > 0 and (query.data_ptr() % 16 or query.stride(3) != 1 or any(query.stride(i) <= 0 or query.stride(i) % 8 for i in (0, 1))):
        query = query.contiguous()   # the prefix's kernel copies rows in 16-byte pieces
        if query.data_ptr() % 16:
            query = query.clone()

    p = _lib.CacheDecodeParams()
    p.struct_size = C.sizeof(_lib.CacheDecodeParams)
    p.dtype = ops._DTYPE_CODE[query.dtype]
    p.device = dev = ops._device_index(query)
    p.page_size = page_size
    p.q, p.out = query.data_ptr(), out.data_ptr()
    p.q_stride[:] = [query.stride(i) for i in (0, 1, 3)]
    p.out_stride[:] = [out.stride(i) for i in (0, 1, 3)]
    if lse is not None:
        p.lse = lse.data_ptr()
        p.lse_stride[:] = lse.stride()[:2]
    p.k_pages, p.v_pages = k_pages.data_ptr(), v_pages.data_ptr()
    p.k_pages_stride[:] = _order(k_pages, hd, rd)
    p.v_pages_stride[:] = _order(v_pages, hd, rd)
    if quantised:
        p.k_scales, p.v_scales = k_scales.data_ptr(), v_scales.data_ptr()
        p.k_scales_stride[:] = _order(k_scales, hd, rd)
        p.v_scales_stride[:] = _order(v_scales, hd, rd)
    p.B, p.Hq, p.Hkv, p.D = B, Hq, Hkv, D
    p.scale = float(1.0 / math.sqrt(D) if scale is None else scale)
    p.n_pages = k_pages.shape[0]
    p.kv_lens = kv_lens.data_ptr()
    p.block_table_stride = block_table.shape[1]
    if block_table.shape[1]:
        p.block_table = block_table.data_ptr()
    p.prefix_len = prefix_len
    if prefix_len:
        p.prefix_table = prefix_table.data_ptr()
    p.kv_chunk = int(kv_chunk)
    p.status = ops._status_word(dev).data_ptr()
    if not quantised and prefix_len == 0:
        return ops.paged_decode(query, k_pages, v_pages, block_table, kv_lens, scale=scale, layout=layout, out=out, lse=lse,
                                need_lse=need_lse, kv_chunk=kv_chunk)
    lib = _lib.load()
    plan = _lib.Plan()
    plan.struct_size = C.sizeof(_lib.Plan)
    rc = lib.b200_sdpa_cache_decode_plan(C.byref(p), C.byref(plan))
    if rc != _lib.OK:
        raise RuntimeError(f"b200_sdpa_cache_decode_plan: {_lib.strerror(rc)}")
    # scratch of this call's own: the interpreter lock is not held while its launches are queued, and another thread's, on the same
    # stream, may come between them.  The block goes back to the (stream-ordered) allocator when they have been.
    ws = torch.empty(max(int(plan.workspace_bytes), 16), dtype=torch.uint8, device=query.device)
    p.workspace = ws.data_ptr()
    p.workspace_bytes = ws.numel()
    _launch("b200_sdpa_cache_decode", p)
    return out, lse

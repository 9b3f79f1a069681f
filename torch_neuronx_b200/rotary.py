"""Rotary position embedding of queries and keys, with one to four position axes, forward and backward.

A multimodal prompt gives every token a position on several axes (time, height, width); each axis turns its own
section of the frequency pairs.  With one axis this is the usual rotary embedding.  The decode kernels rotate an
appended row themselves (:func:`ops.paged_decode` with ``rope_cos``); prompts, training steps and 8-bit caches use this.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch
from torch.autograd import forward_ad

from . import _lib, ops

_MAX_AXES = 4


def rotary_embedding(
    query: torch.Tensor,
    key: Optional[torch.Tensor],
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    *,
    sections: Optional[Sequence[int]] = None,
    interleaved: bool = False,
):
    """``(query, key)`` rotated by their positions, in new tensors of the same layout; ``key`` may be ``None``.

    ``query`` is ``(B, Hq, L, D)`` and ``key`` ``(B, Hkv, L, D)``, any strides, fp32, fp16 or bf16, ``B`` at most 65535.  ``inv_freq`` is a
    contiguous fp32 or fp64 vector of ``R / 2`` frequencies (``R <= D``, even; elements behind ``R`` are copied).  ``positions`` is
    int32 or int64, ``(axes, B, L)``, or ``(B, L)`` or ``(L,)`` for one axis; extents of 1 are broadcast.  ``sections``
    says how many consecutive pairs belong to each axis (their sum is ``R / 2``).  Pair ``i`` is elements ``(i, i + R / 2)``, or
    ``(2 i, 2 i + 1)`` when ``interleaved``, and is turned by ``positions[axis of i] * inv_freq[i]``, an angle that is formed in
    64 bits; the rest is computed in 32 and rounded once.  Gradients and forward-mode tangents flow to ``query`` and ``key``, none to ``inv_freq``; a trace cannot record
    the call.  A backward pass
    captured into a CUDA graph is refused while an eager graph that was built on the default stream still holds one of its leaves."""
    if _lib.native is not None and not torch.compiler.is_compiling():
        got = _lib.native.rotary(query, key, positions, inv_freq, sections, interleaved)
        if got is not None:
            return got
    ops._check_visible("rotary_embedding", inv_freq)
    args = _check(query, key, positions, inv_freq, sections)
    tangents = [None if x is None else forward_ad.unpack_dual(x).tangent for x in (query, key)]
    if any(t is not None for t in tangents):
        return _forward_mode(query, key, tangents, *args, interleaved)
    wants = torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad))
    if wants:
        return _Rotary.apply(query, key, *args, bool(interleaved), False)
    return _rotate(query, key, *args, bool(interleaved), False)


def _forward_mode(query, key, tangents, positions, inv_freq, sections, interleaved):
    """A rotation is linear: the tangents are rotated like the tensors that carry them."""
    got = []
    for x, t in zip((query, key), tangents):
        if x is None:
            got.append(None)
            continue
        y, _ = rotary_embedding(forward_ad.unpack_dual(x).primal, None, positions, inv_freq, sections=sections, interleaved=interleaved)
        if t is not None:
            y = forward_ad.make_dual(y, rotary_embedding(t, None, positions, inv_freq, sections=sections, interleaved=interleaved)[0])
        got.append(y)
    return tuple(got)


def _check(query, key, positions, inv_freq, sections):
    """The arguments' rules; returns ``(positions as (axes, B, L), inv_freq, sections)``."""
    if query.dim() != 4 or (key is not None and key.dim() != 4):
        raise RuntimeError("rotary_embedding: query and key must be 4-D (B, H, L, D)")
    if not query.is_cuda:
        raise ValueError(f"Expected CUDA device, got {query.device}")
    if query.dtype not in ops._DTYPE_CODE:
        raise RuntimeError("rotary_embedding: query must be float32, float16 or bfloat16")
    B, _, L, D = query.shape
    if key is not None and (key.dtype != query.dtype or key.device != query.device or key.shape[0] != B or key.shape[2:] != query.shape[2:]):
        raise RuntimeError("rotary_embedding: key must share the query's batch, length, head dim, dtype and device")
    if max(query.shape) > ops._MOST or (key is not None and key.shape[1] > ops._MOST):
        raise RuntimeError("rotary_embedding: extents are counted in 32 bits")
    if positions.dtype not in (torch.int32, torch.int64) or positions.device != query.device or not 1 <= positions.dim() <= 3:
        raise RuntimeError("rotary_embedding: positions must be an int32 or int64 tensor (axes, B, L), (B, L) or (L,) on the query's device")
    axes = positions.shape[0] if positions.dim() == 3 else 1
    try:
        positions = positions.expand(axes, B, L)
    except RuntimeError:
        raise RuntimeError(f"rotary_embedding: positions {tuple(positions.shape)} do not broadcast to ({axes}, {B}, {L})") from None
    if inv_freq.dtype not in (torch.float32, torch.float64) or inv_freq.dim() != 1 or inv_freq.device != query.device or not inv_freq.is_contiguous():
        raise RuntimeError("rotary_embedding: inv_freq must be a contiguous float32 or float64 vector on the query's device")
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("rotary_embedding: no gradient flows to inv_freq, which requires one; detach it")
    pairs = inv_freq.shape[0]
    if pairs < 1 or 2 * pairs > D:
        raise RuntimeError(f"rotary_embedding: inv_freq has {pairs} frequencies, the head dim {D} has room for 1 to {D // 2}")
    if sections is None:
        if axes != 1:
            raise RuntimeError("rotary_embedding: several position axes need sections")
        sections = (pairs,)
    sections = tuple(int(n) for n in sections)
    if not 1 <= axes <= _MAX_AXES or len(sections) != axes or any(n < 0 for n in sections) or sum(sections) != pairs:
        raise RuntimeError(f"rotary_embedding: sections {sections} must give each of the {axes} axes (at most {_MAX_AXES}) its pairs, {pairs} in all")
    return positions, inv_freq, sections


def _rotate(query, key, positions, inv_freq, sections, interleaved: bool, inverse: bool):
    xs = (query,) if key is None else (query, key)
    ys = tuple(ops.alloc_like_query(x, x.shape) for x in xs)
    if any(x.numel() == 0 for x in xs):
        # nothing of one of them to turn: the other alone
        if len(xs) == 2 and xs[0].numel() != 0:
            return _rotate(query, None, positions, inv_freq, sections, interleaved, inverse)[0], ys[1]
        if len(xs) == 2 and xs[1].numel() != 0:
            return ys[0], _rotate(key, None, positions, inv_freq, sections, interleaved, inverse)[0]
        return ys if key is not None else (ys[0], None)
    p = _lib.RotaryParams()
    p.struct_size = C.sizeof(_lib.RotaryParams)
    p.dtype = ops._DTYPE_CODE[query.dtype]
    p.device = ops._device_index(query)
    p.inverse = 1 if inverse else 0
    for i, (x, y) in enumerate(zip(xs, ys)):
        p.x[i], p.y[i] = x.data_ptr(), y.data_ptr()
        p.x_stride[i][:] = x.stride()
        p.y_stride[i][:] = y.stride()
        p.heads[i] = x.shape[1]
    p.B, p.L, p.D = query.shape[0], query.shape[2], query.shape[3]
    p.rot = 2 * inv_freq.shape[0]
    p.axes = len(sections)
    p.interleaved = 1 if interleaved else 0
    p.section[: len(sections)] = sections
    p.positions, p.inv_freq = positions.data_ptr(), inv_freq.data_ptr()
    p.pos_stride[:] = positions.stride()
    p.positions_i64 = 1 if positions.dtype == torch.int64 else 0
    p.inv_freq_f64 = 1 if inv_freq.dtype == torch.float64 else 0
    p.status = ops._status_word(p.device).data_ptr()
    lib = _lib.load()
    rc = lib.b200_sdpa_rotary(C.byref(p), C.c_void_p(torch.cuda.current_stream(p.device).cuda_stream))
    if rc != _lib.OK:
        raise RuntimeError(f"b200_sdpa_rotary: {_lib.strerror(rc)}")
    return ys if key is not None else (ys[0], None)


class _Rotary(torch.autograd.Function):
    """A rotation's gradient is the rotation by the opposite angle, itself differentiable."""

    @staticmethod
    def forward(ctx, query, key, positions, inv_freq, sections, interleaved, inverse):
        ctx.save_for_backward(positions, inv_freq)
        ctx.rest = (sections, interleaved, inverse)
        ctx.set_materialize_grads(False)
        return _rotate(query, key, positions, inv_freq, sections, interleaved, inverse)

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        if _lib.native is not None:
            _lib.native.check_leaf_streams()
        positions, inv_freq = ctx.saved_tensors
        sections, interleaved, inverse = ctx.rest
        want_q = grad_query is not None and ctx.needs_input_grad[0]
        want_k = grad_key is not None and ctx.needs_input_grad[1]
        got_q = got_k = None
        if want_q:
            got_q, got_k = _Rotary.apply(grad_query, grad_key if want_k else None, positions, inv_freq, sections, interleaved, not inverse)
        elif want_k:
            got_k, _ = _Rotary.apply(grad_key, None, positions, inv_freq, sections, interleaved, not inverse)
        return got_q, got_k, None, None, None, None, None

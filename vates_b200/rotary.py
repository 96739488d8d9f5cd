"""Rotary positions with several axes (time, height, width of images and video)
for tokens whose positions are given (``vb_rotate_axes``), with the RMS norm of
q and k that some models have before it.

Attention over a cache does not care in which row a key lies, so once rows have
been evicted (:meth:`vates_b200.kv8.PagedKV8Cache.evict`) the position of a new
token is no longer the row it is written to: it is given here instead.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from ._lib import VbRotateArgs, check, lib
from .pool import current_device, current_stream, on_device

# Argument structures without pointers, and the host tables they refer to, by layout: the
# types, shapes and strides of a call's tensors and its other arguments, checked once.
_LAYOUTS: dict = {}


def pair_axes(sections, interleaved: bool = False) -> tuple:
    """The axis of every rotated pair from the number of pairs per axis: one
    section after another, or, ``interleaved``, dealt out in turn (0, 1, 2, 0,
    1, 2, ...) for as long as an axis has pairs left."""
    sections = [int(n) for n in sections]
    if any(n < 0 for n in sections):
        raise ValueError(f"sections={sections}: pairs per axis, none negative")
    if not interleaved:
        return tuple(a for a, n in enumerate(sections) for _ in range(n))
    return tuple(a for i in range(max(sections, default=0))
                 for a, n in enumerate(sections) if i < n)


def _check(t: torch.Tensor, what: str, shape):
    # (an empty tensor's strides may be anything)
    if t.dtype != torch.bfloat16 or t.shape != shape \
            or (t.numel() and t.stride()[-1:] not in ((1,), ())):
        raise ValueError(f"{what}: bfloat16 {tuple(shape)} with contiguous dims is needed, got "
                         f"{t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def _layout(key, q, k, positions, axes, base, eps, q_norm, k_norm, q_out, k_out):
    """The arguments of a call but its tensors' addresses."""
    B, Hq, L, D = q.shape
    _check(q, "q", q.shape)
    _check(k, "k", (B, k.shape[1], L, D))
    for t, shape, what in ((q_norm, (D,), "q_norm"), (k_norm, (D,), "k_norm"),
                           (q_out, q.shape, "q_out"), (k_out, k.shape, "k_out")):
        if t is not None:
            _check(t, what, shape)
    if positions.dtype != torch.int32 or positions.dim() != 3 or positions.shape[1:] != (B, L) \
            or not positions.is_contiguous():
        raise ValueError(f"positions: contiguous int32 [axes, {B}, {L}] is needed, got "
                         f"{positions.dtype} {tuple(positions.shape)}")
    if not 1.0 < base < math.inf:
        raise ValueError(f"base={base}: a finite number above 1 is needed")
    n, count = len(axes), positions.shape[0]
    if n > 128 or n % 8 or n == 0 or any(not 0 <= a < count for a in axes):
        raise ValueError(f"axes: one axis per pair (of {count} in positions), a multiple of 8 "
                         f"pairs and at most 128, got {n} pairs of the axes {sorted(set(axes))}")
    axis = (C.c_uint8 * n)(*axes)
    turns = (C.c_double * n)(*[base ** (-i / n) / (2.0 * math.pi) for i in range(n)])
    dense = lambda h: (h * L * D, L * D, D)
    strides = [(C.c_int64 * 3)(*x[:3]) for x in
               (q.stride(), k.stride(), dense(Hq) if q_out is None else q_out.stride(),
                dense(k.shape[1]) if k_out is None else k_out.stride())]
    a = VbRotateArgs(None, None, None, None, None, None, *strides, None, C.cast(turns, C.c_void_p),
                     C.cast(axis, C.c_void_p), eps, B, L, Hq, k.shape[1], D, 2 * n, count)
    if len(_LAYOUTS) > 4096:
        _LAYOUTS.clear()
    _LAYOUTS[key] = got = (bytes(a), axis, turns)
    return got


def rotate_axes(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, axes,
                base: float = 10_000_000.0, q_norm=None, k_norm=None, eps: float = 1e-6,
                q_out=None, k_out=None, stream=None):
    """``(q, k)`` with the first ``2 len(axes)`` dims of every row rotated: pair
    ``(i, i + len(axes))`` of token ``t`` of sequence ``b`` by the angle
    ``positions[axes[i], b, t] * base ** (-i / len(axes))``.

    ``q`` bf16 ``[batch, heads, L, dim]`` and ``k`` ``[batch, kv_heads, L, dim]``
    (any strides with contiguous dims, a projection's layout for one); ``dim`` a
    multiple of 16, at most 256. ``positions`` int32 ``[axes, batch, L]``, any
    values; ``axes`` the axis of every pair (:func:`pair_axes`), a multiple of 8
    pairs. ``q_norm``, ``k_norm`` bf16 ``[dim]``: rows are RMS-normalised and
    multiplied by it first. Float32 throughout, rounded to bf16 once. Results are
    new contiguous tensors, or ``q_out`` and ``k_out``, which may be ``q`` and
    ``k`` themselves but must not overlap them in any other way, nor hold two rows in
    one place (an expanded tensor)."""
    dev = q.get_device()
    # with it as the current stream, results belong to it
    if dev >= 0 and (stream is not None or current_device() != dev):
        with on_device(q.device, stream):
            return rotate_axes(q, k, positions, axes, base, q_norm, k_norm, eps, q_out, k_out)
    if q.dim() != 4 or k.dim() != 4 or dev < 0:
        raise ValueError("q, k: CUDA [batch, heads, L, dim] are needed, got "
                         f"{tuple(q.shape)} and {tuple(k.shape)} on {q.device}")
    others = [t for t in (k, positions, q_norm, k_norm, q_out, k_out) if t is not None]
    for t in others:
        if t.get_device() != dev:
            raise ValueError(f"a tensor on {t.device}, q on cuda:{dev}")
    if q.stride(3) != 1 and q.numel():
        q = q.contiguous()
    if k.stride(3) != 1 and k.numel():
        k = k.contiguous()
    if type(axes) is not tuple:
        axes = tuple(int(a) for a in axes)
    key = (q.dtype, q.shape, q.stride(), axes, base, eps,
           *[x for t in others for x in (t.dtype, t.shape, t.stride())],
           q_norm is None, k_norm is None, q_out is None, k_out is None)
    layout = _LAYOUTS.get(key)
    if layout is None:
        layout = _layout(key, q, k, positions, axes, base, eps, q_norm, k_norm, q_out, k_out)
    if q_out is None:
        q_out = q.new_empty(q.shape)
    if k_out is None:
        k_out = k.new_empty(k.shape)
    a = VbRotateArgs.from_buffer_copy(layout[0])
    a.q, a.k, a.q_out, a.k_out = q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr()
    a.positions = positions.data_ptr()
    if q_norm is not None:
        a.q_norm = q_norm.data_ptr()
    if k_norm is not None:
        a.k_norm = k_norm.data_ptr()
    check(lib.vb_rotate_axes(C.byref(a), current_stream(dev)), "vb_rotate_axes")
    return q_out, k_out


__all__ = ["pair_axes", "rotate_axes"]

"""Paged 8-bit KV cache on B200: writing, reading back and attention.

A pool of pages holds int8 codes ``[pages, kv_heads, page, head_dim]`` for K
and for V with one float32 scale per page and head (``value = code * scale``);
a table ``[batch, max_pages]`` names the pool page of every ``page``
consecutive positions of a sequence. Positions and lengths are device tensors,
so a step that writes and attends can be captured in a CUDA graph, which then
owns the scratch of its calls (:mod:`vates_b200.scratch`).

Half the bytes of a bf16 cache, several sequences of different lengths, any
number of query heads per key/value head and head sizes 64, 128 and 256; the
IsoQuant cache (:mod:`vates_b200.quant_kv`) is smaller still, for one head
size and one common length. The kernels are in ``libvates_b200`` (no
fallback).
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import (VbKv8AppendArgs, VbKv8AttnArgs, VbKv8Cache, VbKv8ReadArgs, check, lib)
from .pool import current_device, current_stream, on_device, ptr, status_ptr
from .scratch import Scratch

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
# partial results of the key ranges; one for the caches of all layers, whose
# attention on a stream runs one after another
_scratch = Scratch(_lib.VB_KV8_ATTN_WORKSPACE_HEAD)


def _rows(t: torch.Tensor, what: str, shape, device: int) -> torch.Tensor:
    """``t`` as bf16 rows on the GPU with contiguous dims (other strides stay)."""
    if t.dtype != torch.bfloat16 or t.get_device() != device:
        raise ValueError(f"{what}: a bfloat16 tensor on cuda:{device} is needed, got {t.dtype} on "
                         f"{t.device}")
    if t.shape != shape:
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t if t.stride(3) == 1 else t.contiguous()


def _ints(t: torch.Tensor | None, what: str, batch: int, device: int) -> int | None:
    """Device pointer of a contiguous int32 ``[batch]`` tensor."""
    if t is None:
        return None
    if t.dtype != torch.int32 or t.get_device() != device or t.numel() != batch \
            or not t.is_contiguous():
        raise ValueError(f"{what}: a contiguous int32 tensor of {batch} values on cuda:{device} "
                         f"is needed, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


_STRIDES: dict = {}


def _strides(t: torch.Tensor):
    """Strides of batch, head and row as the C array (made once per layout)."""
    s = t.stride()
    a = _STRIDES.get(s)
    if a is None:
        if len(_STRIDES) > 4096:
            _STRIDES.clear()
        a = _STRIDES[s] = (C.c_int64 * 3)(*s[:3])
    return a


class PagedKV8Cache:
    """One layer's cache. The tensors are the caller's (or :meth:`empty`'s) and
    may be shared between caches with different tables; a page that is written
    must belong to one sequence only. Scales are finite and not negative. The
    table may be edited in place or replaced (:attr:`page_table`) between calls;
    a CUDA graph keeps reading the one it was captured with."""

    def __init__(self, k_codes, v_codes, k_scales, v_scales, page_table):
        if k_codes.dim() != 4:
            raise ValueError("codes are [pages, kv_heads, page, head_dim]")
        pages, heads, page, dim = k_codes.shape
        self.device = k_codes.device
        if page not in PAGE_SIZES or dim not in HEAD_DIMS:
            raise ValueError(f"page of {page} rows (one of {PAGE_SIZES}), head_dim {dim} "
                             f"(one of {HEAD_DIMS})")
        for t, shape, dt in ((k_codes, k_codes.shape, torch.int8),
                             (v_codes, k_codes.shape, torch.int8),
                             (k_scales, (pages, heads), torch.float32),
                             (v_scales, (pages, heads), torch.float32)):
            if tuple(t.shape) != tuple(shape) or t.dtype != dt or not t.is_contiguous() \
                    or not t.is_cuda or t.device != self.device:
                raise ValueError(f"cache tensor: contiguous CUDA {dt} {tuple(shape)} is needed, "
                                 f"got {t.dtype} {tuple(t.shape)} on {t.device}")
        self.k_codes, self.v_codes = k_codes, v_codes
        self.k_scales, self.v_scales = k_scales, v_scales
        self.pages, self.kv_heads, self.page, self.head_dim = pages, heads, page, dim
        self._index = k_codes.get_device()
        self.page_table = page_table

    @property
    def page_table(self) -> torch.Tensor:
        return self._table

    @page_table.setter
    def page_table(self, t: torch.Tensor):
        if t.dim() != 2 or t.dtype != torch.int32 or not t.is_contiguous() \
                or t.device != self.device:
            raise ValueError("page_table: a contiguous int32 [batch, max_pages] tensor on "
                             f"{self.device} is needed, got {t.dtype} {tuple(t.shape)} on "
                             f"{t.device}")
        self._table = t
        self.batch = t.shape[0]
        # argument structures with the cache filled in, copied for each call
        c = VbKv8Cache(self.k_codes.data_ptr(), self.v_codes.data_ptr(),
                       self.k_scales.data_ptr(), self.v_scales.data_ptr(), t.data_ptr(),
                       self.pages, self.kv_heads, self.page, self.head_dim, *t.shape)
        self._append_args = bytes(VbKv8AppendArgs(c))
        self._read_args = bytes(VbKv8ReadArgs(c))
        self._attn_args = bytes(VbKv8AttnArgs(c))
        self._need = {}  # workspace bytes by (q_heads, L)

    @classmethod
    def empty(cls, pages: int, kv_heads: int, head_dim: int, batch: int, max_pages: int,
              page: int = 64, device="cuda"):
        """A cache of ``pages`` unused pages whose table names none yet (-1)."""
        codes = [torch.zeros((pages, kv_heads, page, head_dim), dtype=torch.int8, device=device)
                 for _ in range(2)]
        scales = [torch.zeros((pages, kv_heads), dtype=torch.float32, device=device)
                  for _ in range(2)]
        table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        return cls(*codes, *scales, table)

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in
                   (self.k_codes, self.v_codes, self.k_scales, self.v_scales))

    # ------------------------------------------------------------------ write
    def append(self, keys, values, pos, counts=None, pos_add: int = 0, status=None, stream=None):
        """Quantise rows as they are written: row ``i < counts[b]`` (all ``n``
        without ``counts``) of ``keys``/``values`` bf16 ``[batch, kv_heads, n,
        head_dim]`` goes to position ``pos[b] + pos_add + i``. A page's scale is
        max|x| / 127 over the rows it received; when new rows raise it, the
        page's older codes are rounded again under the new scale. Writing again
        from an earlier position (rows taken back) keeps the scale that the
        rows taken back gave the page, unless it starts at the page's first
        row. Rows past the
        table set VB_STATUS_BOUNDS in ``status`` and are dropped; an infinity is
        stored as the page's largest value, a NaN as 0, with
        VB_STATUS_NONFINITE."""
        # with it as the current stream, copies are made on it
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.append(keys, values, pos, counts, pos_add, status)
        B, n = self.batch, keys.shape[2] if keys.dim() == 4 else -1
        shape = (B, self.kv_heads, n, self.head_dim)
        dev = self._index
        keys, values = _rows(keys, "keys", shape, dev), _rows(values, "values", shape, dev)
        a = VbKv8AppendArgs.from_buffer_copy(self._append_args)
        a.keys, a.values = keys.data_ptr(), values.data_ptr()
        a.k_strides, a.v_strides = _strides(keys), _strides(values)
        a.pos, a.counts = _ints(pos, "pos", B, dev), _ints(counts, "counts", B, dev)
        a.pos_add, a.n = pos_add, n
        if status is not None:
            a.status = status_ptr(status, dev)
        check(lib.vb_kv8_append(C.byref(a), current_stream(dev)), "vb_kv8_append")

    # -------------------------------------------------------------- read back
    def read(self, lens, n: int, start=None, status=None, stream=None):
        """``(keys, values)`` bf16 ``[batch, kv_heads, n, head_dim]``: the rows
        at positions ``start[b] + i`` (``start`` None: 0), zero from ``lens[b]``
        on."""
        # with it as the current stream, results belong to it
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.read(lens, n, start, status)
        B, dev = self.batch, self._index
        keys = self.k_codes.new_empty((B, self.kv_heads, n, self.head_dim), dtype=torch.bfloat16)
        values = torch.empty_like(keys)
        a = VbKv8ReadArgs.from_buffer_copy(self._read_args)
        a.lens, a.start = _ints(lens, "lens", B, dev), _ints(start, "start", B, dev)
        a.keys, a.values = keys.data_ptr(), values.data_ptr()
        a.n = n
        if status is not None:
            a.status = status_ptr(status, dev)
        check(lib.vb_kv8_read(C.byref(a), current_stream(dev)), "vb_kv8_read")
        return keys, values

    # -------------------------------------------------------------- attention
    def attend(self, q, lens, q_lens=None, len_add: int = 0, scale: float | None = None,
               causal: bool = True, out=None, return_lse: bool = False, status=None, stream=None,
               workspace=None):
        """``softmax(scale * q K^T) V`` over the ``lens[b] + len_add`` keys of
        every sequence. ``q`` bf16 ``[batch, q_heads, L, head_dim]``; query row
        ``i < q_lens[b]`` (``L`` without) is the sequence's row ``keys - q_lens
        + i`` and with ``causal`` sees the keys up to itself. Rows that see
        nothing, and rows from ``q_lens[b]`` on, are zero (log-sum-exp -inf).
        Returns bf16 ``[batch, q_heads, L, head_dim]``, with ``return_lse``
        also float32 ``[batch, q_heads, L]`` (natural log). ``workspace``: the
        caller's scratch (:meth:`attend_workspace_size` bytes, uint8, zeros
        before its first call) for calls that never overlap, in graphs or not;
        without it a call finds its own."""
        # with it as the current stream, results belong to it
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.attend(q, lens, q_lens, len_add, scale, causal, out, return_lse,
                                   status, workspace=workspace)
        B, D, dev = self.batch, self.head_dim, self._index
        if q.dim() != 4:
            raise ValueError(f"q: [batch, q_heads, L, head_dim] is needed, got {tuple(q.shape)}")
        Hq, L = q.shape[1], q.shape[2]
        q = _rows(q, "q", (B, Hq, L, D), dev)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif out.shape != q.shape or out.dtype != torch.bfloat16 or not out.is_contiguous() \
                or out.get_device() != dev:
            raise ValueError(f"out: contiguous bfloat16 of q's shape on cuda:{dev} is needed, got "
                             f"{out.dtype} {tuple(out.shape)} on {out.device}")
        lse = q.new_empty((B, Hq, L), dtype=torch.float32) if return_lse else None
        a = VbKv8AttnArgs.from_buffer_copy(self._attn_args)
        a.q, a.q_strides = q.data_ptr(), _strides(q)
        a.lens, a.q_lens = _ints(lens, "lens", B, dev), _ints(q_lens, "q_lens", B, dev)
        a.out, a.lse = out.data_ptr(), ptr(lse)
        if status is not None:
            a.status = status_ptr(status, dev)
        a.scale = D ** -0.5 if scale is None else scale
        a.q_heads, a.L, a.len_add, a.causal = Hq, L, len_add, causal
        need = self._need.get((Hq, L))
        if need is None:
            need = self._need[Hq, L] = lib.vb_kv8_attn_workspace_size(C.byref(a))
        st = current_stream(dev)
        if workspace is not None:
            if workspace.dtype != torch.uint8 or workspace.get_device() != dev \
                    or not workspace.is_contiguous():
                raise ValueError(f"workspace: contiguous uint8 on cuda:{dev} is needed, got "
                                 f"{workspace.dtype} on {workspace.device}")
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
        elif need:
            ws = _scratch.get(need, self.device, st)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.vb_kv8_attn(C.byref(a), st), "vb_kv8_attn")
        return (out, lse) if return_lse else out

    def attend_workspace_size(self, q_heads: int, L: int) -> int:
        """Bytes of scratch that :meth:`attend` needs for ``L`` rows of
        ``q_heads`` heads with the present page table."""
        a = VbKv8AttnArgs.from_buffer_copy(self._attn_args)
        a.q_heads, a.L = q_heads, L
        return lib.vb_kv8_attn_workspace_size(C.byref(a))


__all__ = ["PagedKV8Cache"]

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
from ._lib import (VbKv8AppendArgs, VbKv8AttnArgs, VbKv8Cache, VbKv8EvictArgs, VbKv8ReadArgs,
                   VbKv8SharedArgs, VbKv8WeighArgs, check, lib)
from .pool import current_device, current_stream, on_device, ptr, status_ptr
from .scratch import Scratch

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128, 256)
# partial results of the key ranges; one for the caches of all layers, whose
# attention on a stream runs one after another
_scratch = Scratch(_lib.VB_KV8_ATTN_WORKSPACE_HEAD)
_lists = Scratch(16)  # what calls of weigh and evict make for themselves


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


class SharedPrefix:
    """Which sequences of a batch share the rows they begin with: ``groups`` of
    ``(first, count, rows)``, the ``count`` sequences from ``first`` on whose first
    ``rows`` rows (whole pages) are the same pool pages in the page table of each of
    them, as far as it holds that many keys; in order, each sequence in one group at
    most. For :meth:`PagedKV8Cache.attend_shared` of ``cache`` and of every other one
    with its batch, page size and device, as those of the other layers. A CUDA graph
    keeps to the groups it was captured with, and needs this object for as long as it is
    replayed.

    Sharing costs two more kernels, so a call whose groups save fewer than ``least``
    bytes of K and V (:attr:`groups`' rows, for all but one of their sequences) attends
    every sequence by itself; without ``least``, where that was measured to be faster."""

    def __init__(self, cache: "PagedKV8Cache", groups, least: int | None = None):
        self.batch, self.page, self.device = cache.batch, cache.page, cache.device
        self.groups = tuple((int(f), int(n), int(rows)) for f, n, rows in groups)
        end, most = 0, cache.page_table.shape[1] * self.page
        for first, count, rows in self.groups:
            if first < end or count < 1 or first + count > self.batch or rows < self.page \
                    or rows % self.page or rows > most:
                raise ValueError(f"group {(first, count, rows)}: sequences of {self.batch} in order,"
                                 f" rows in whole pages of {self.page}, at most {most}")
            end = first + count
        # a group of one gains nothing: its sequence is attended as a whole
        kept = [g for g in self.groups if g[1] > 1]
        group_of, start = [-1] * self.batch, [0] * self.batch
        for g, (first, count, rows) in enumerate(kept):
            group_of[first:first + count] = [g] * count
            start[first:first + count] = [rows] * count
        words = [x for f, n, rows in kept for x in (f, n, 0, rows)]
        words += [x for b, s in enumerate(start) for x in (b, 1, s, 0x7fffffff)]
        # segments, then the groups of sequences
        self._words = torch.tensor(words + group_of, dtype=torch.int32).to(self.device)
        self._segments = self._words.data_ptr()
        self._group_of = self._segments + 4 * len(words)
        self._stream = current_stream(self._words.get_device())  # whose memory _words is
        self._host = (C.c_int32 * (3 * len(kept)))(*[x for g in kept for x in g])
        self._count = len(kept)
        self._longest = max([rows // self.page for _, _, rows in kept], default=0)
        if least is not None and least < 0:
            raise ValueError(f"least={least}: a number of bytes")
        self._least = -1 if least is None else least
        # workspace bytes, and whether groups are attended as such, by (cache layout, q_heads, L)
        self._need: dict = {}
        self._shares: dict = {}


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
        self._weigh_args = bytes(VbKv8WeighArgs(c))
        self._evict_args = bytes(VbKv8EvictArgs(c))
        self._shared_args = bytes(VbKv8SharedArgs(VbKv8AttnArgs(c)))
        self._need = {}  # workspace bytes by (q_heads, L), of others by name and sizes

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
        caller's scratch (:meth:`attend_workspace_size` bytes, uint8, 32-byte aligned, zeros
        before its first call) for calls that never overlap, in graphs or not;
        without it a call finds its own."""
        # with it as the current stream, results belong to it
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.attend(q, lens, q_lens, len_add, scale, causal, out, return_lse,
                                   status, workspace=workspace)
        dev = self._index
        a = VbKv8AttnArgs.from_buffer_copy(self._attn_args)
        q, out, lse = self._attn_fill(a, q, lens, q_lens, len_add, scale, causal, out, return_lse,
                                      status)
        Hq, L = a.q_heads, a.L
        need = self._need.get((Hq, L))
        if need is None:
            need = self._need[Hq, L] = lib.vb_kv8_attn_workspace_size(C.byref(a))
        st = current_stream(dev)
        self._attn_workspace(a, workspace, need, st)
        check(lib.vb_kv8_attn(C.byref(a), st), "vb_kv8_attn")
        return (out, lse) if return_lse else out

    def attend_shared(self, q, lens, shared: SharedPrefix, q_lens=None, len_add: int = 0,
                      scale: float | None = None, causal: bool = True, out=None,
                      return_lse: bool = False, status=None, stream=None, workspace=None):
        """What :meth:`attend` gives for a batch whose sequences share the rows they
        begin with in groups (:class:`SharedPrefix`): those are read, and multiplied,
        once for the query rows of all sequences of a group, where that saves enough.
        ``lens`` and positions count the shared rows, as in every other call.
        ``workspace``: as in :meth:`attend`, of :meth:`shared_workspace_size` bytes."""
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.attend_shared(q, lens, shared, q_lens, len_add, scale, causal, out,
                                          return_lse, status, workspace=workspace)
        if q.dim() == 4 and not self._shares(shared, q.shape[1], q.shape[2]):
            return self.attend(q, lens, q_lens, len_add, scale, causal, out, return_lse, status,
                               workspace=workspace)
        s, dev = self._shared_fill(shared), self._index
        q, out, lse = self._attn_fill(s.attn, q, lens, q_lens, len_add, scale, causal, out,
                                      return_lse, status)
        st = current_stream(dev)
        self._attn_workspace(s.attn, workspace, self._shared_need(shared, s), st)
        if st != shared._stream:  # a plan that is let go now is read by the kernels all the same
            shared._words.record_stream(torch.cuda.current_stream(dev))
        check(lib.vb_kv8_attn_shared(C.byref(s), st), "vb_kv8_attn_shared")
        return (out, lse) if return_lse else out

    def shared_workspace_size(self, shared: SharedPrefix, q_heads: int, L: int) -> int:
        """Bytes of scratch that :meth:`attend_shared` needs for ``L`` rows of
        ``q_heads`` heads with the present page table."""
        if not self._shares(shared, q_heads, L):
            return self.attend_workspace_size(q_heads, L)
        s = self._shared_fill(shared)
        s.attn.q_heads, s.attn.L = q_heads, L
        return self._shared_need(shared, s)

    def _shares(self, shared: SharedPrefix, q_heads: int, L: int) -> bool:
        """Whether the groups of ``shared`` are attended as such."""
        if shared.batch != self.batch or shared.page != self.page \
                or shared.device != self.device or shared._longest > self._table.shape[1]:
            raise ValueError(f"shared: groups of {shared.batch} sequences in pages of {shared.page} "
                             f"on {shared.device}, up to {shared._longest}; the cache has "
                             f"{self.batch} in pages of {self.page} on {self.device}, "
                             f"{self._table.shape[1]} each")
        key = (self.kv_heads, self.head_dim, self._table.shape[1], q_heads, L)
        shares = shared._shares.get(key)
        if shares is None:
            shares = False
            if shared._count:
                s = self._shared_fill(shared)
                s.attn.q_heads, s.attn.L = q_heads, L
                shares = bool(lib.vb_kv8_attn_shares(C.byref(s)))
            shared._shares[key] = shares
        return shares

    def _shared_fill(self, shared: SharedPrefix) -> VbKv8SharedArgs:
        s = VbKv8SharedArgs.from_buffer_copy(self._shared_args)
        s.segments, s.group_of = shared._segments, shared._group_of
        s.host_groups, s.groups = C.addressof(shared._host), shared._count
        s.least = shared._least
        return s

    def _shared_need(self, shared: SharedPrefix, s: VbKv8SharedArgs) -> int:
        key = (self.kv_heads, self.head_dim, self._table.shape[1], s.attn.q_heads, s.attn.L)
        need = shared._need.get(key)
        if need is None:
            need = shared._need[key] = lib.vb_kv8_attn_shared_workspace_size(C.byref(s))
        return need

    def _attn_fill(self, a: VbKv8AttnArgs, q, lens, q_lens, len_add, scale, causal, out,
                   return_lse, status):
        """Checks the arguments of attention and puts them into ``a``."""
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
        a.q, a.q_strides = q.data_ptr(), _strides(q)
        a.lens, a.q_lens = _ints(lens, "lens", B, dev), _ints(q_lens, "q_lens", B, dev)
        a.out, a.lse = out.data_ptr(), ptr(lse)
        if status is not None:
            a.status = status_ptr(status, dev)
        a.scale = D ** -0.5 if scale is None else scale
        a.q_heads, a.L, a.len_add, a.causal = Hq, L, len_add, causal
        return q, out, lse

    def _attn_workspace(self, a: VbKv8AttnArgs, workspace, need: int, st: int):
        dev = self._index
        if workspace is not None:
            if workspace.dtype != torch.uint8 or workspace.get_device() != dev \
                    or not workspace.is_contiguous():
                raise ValueError(f"workspace: contiguous uint8 on cuda:{dev} is needed, got "
                                 f"{workspace.dtype} on {workspace.device}")
            a.workspace, a.workspace_bytes = workspace.data_ptr(), workspace.numel()
        elif need:
            ws = _scratch.get(need, self.device, st)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()

    def attend_workspace_size(self, q_heads: int, L: int) -> int:
        """Bytes of scratch that :meth:`attend` needs for ``L`` rows of
        ``q_heads`` heads with the present page table."""
        a = VbKv8AttnArgs.from_buffer_copy(self._attn_args)
        a.q_heads, a.L = q_heads, L
        return lib.vb_kv8_attn_workspace_size(C.byref(a))

    # --------------------------------------------------------------- eviction
    def _tracked(self, t: torch.Tensor, what: str, dtype, room: int | None) -> int:
        """Pointer of a contiguous ``[batch, kv_heads, room]`` tensor."""
        if t.dtype != dtype or t.get_device() != self._index or t.dim() != 3 \
                or t.shape[0] != self.batch or t.shape[1] != self.kv_heads \
                or (room is not None and t.shape[2] != room) or not t.is_contiguous():
            raise ValueError(f"{what}: contiguous {dtype} [{self.batch}, {self.kv_heads}, "
                             f"{'rows' if room is None else room}] on cuda:{self._index} is needed,"
                             f" got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def weigh(self, q, lse, lens, weights, q_lens=None, new=None, len_add: int = 0,
              scale: float | None = None, causal: bool = True, positions=None, seen=None,
              status=None, stream=None):
        """Add the attention weight that every row receives from the rows of ``q``
        to ``weights`` float32 ``[batch, kv_heads, rows]`` (row ``j`` of a sequence
        at ``j``): over the query heads of a kv head and the query rows that see
        ``j``, the sum of ``exp(scale * q_i . k_j - lse_i)``. ``q``, ``lens``,
        ``q_lens``, ``len_add``, ``scale`` and ``causal`` as in :meth:`attend`,
        ``lse`` its log-sum-exp of the same rows. The last ``new[b]`` rows of a
        sequence (``q_lens[b]`` without it; int32 ``[batch]``) are new to
        ``weights``: they start at 0 and, with ``positions`` int32 of
        ``weights``' shape and ``seen`` int32 ``[batch]``, the sequence's tokens so
        far, take their token's position: ``seen[b] - 1`` for the last of them.
        Rows behind a sequence's last one are left as they are. Query rows whose
        ``lse`` is not finite add nothing (VB_STATUS_NONFINITE in ``status`` but for
        -inf); a sequence longer than ``rows`` is left out with VB_STATUS_BOUNDS."""
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.weigh(q, lse, lens, weights, q_lens, new, len_add, scale, causal,
                                  positions, seen, status)
        B, D, dev = self.batch, self.head_dim, self._index
        if q.dim() != 4:
            raise ValueError(f"q: [batch, q_heads, L, head_dim] is needed, got {tuple(q.shape)}")
        Hq, L = q.shape[1], q.shape[2]
        q = _rows(q, "q", (B, Hq, L, D), dev)
        if lse.dtype != torch.float32 or lse.get_device() != dev or lse.shape != (B, Hq, L) \
                or not lse.is_contiguous():
            raise ValueError(f"lse: contiguous float32 {(B, Hq, L)} on cuda:{dev} is needed, got "
                             f"{lse.dtype} {tuple(lse.shape)} on {lse.device}")
        a = VbKv8WeighArgs.from_buffer_copy(self._weigh_args)
        a.weights = self._tracked(weights, "weights", torch.float32, None)
        a.room = room = weights.shape[2]
        if positions is not None:
            if seen is None:
                raise ValueError("positions need seen, the tokens of every sequence so far")
            a.positions = self._tracked(positions, "positions", torch.int32, room)
            a.seen = _ints(seen, "seen", B, dev)
        a.q, a.q_strides, a.lse = q.data_ptr(), _strides(q), lse.data_ptr()
        a.lens, a.q_lens = _ints(lens, "lens", B, dev), _ints(q_lens, "q_lens", B, dev)
        a.fresh = _ints(new, "new", B, dev)
        if status is not None:
            a.status = status_ptr(status, dev)
        a.scale = D ** -0.5 if scale is None else scale
        a.q_heads, a.L, a.len_add, a.causal = Hq, L, len_add, causal
        need = self._need.get(("weigh", Hq, L, room))
        if need is None:
            need = self._need["weigh", Hq, L, room] = lib.vb_kv8_weigh_workspace_size(C.byref(a))
        st = current_stream(dev)
        if need:
            ws = _lists.get(need, self.device, st)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        check(lib.vb_kv8_weigh(C.byref(a), st), "vb_kv8_weigh")

    def evict(self, weights, lens, keep: int, first: int = 0, recent: int = 0, positions=None,
              status=None, stream=None):
        """Every sequence with more than ``keep`` rows keeps ``keep`` of them, each kv
        head its own: those with the largest ``weights`` (:meth:`weigh`; ties to the
        lower row, NaN last), before them the rows below ``first`` and the
        ``recent`` newest, by ``positions`` (int32 like ``weights``; without it a row's
        number, right until the first eviction). Returns the lengths after it, int32
        ``[batch]``.

        The evicted rows below ``keep`` are replaced, in order, by the kept rows from
        ``keep`` on, in the cache, ``weights`` and ``positions`` alike, so the kept
        rows stay where they are otherwise and the order of rows is no longer the order
        of tokens; ``causal`` attention still hides nothing it should not, as long as
        eviction comes before the step's own rows are appended. A page that receives
        rows takes the largest scale of the pages that its rows come from, and codes of
        a smaller one are rounded again (half a step of the new scale at most). Pages of
        more than one sequence must lie below ``first``. Lengths beyond the page table or
        ``weights`` count as that many rows, and rows to or from a page that is not there
        do not move (VB_STATUS_BOUNDS in ``status``)."""
        if stream is not None or current_device() != self._index:
            with on_device(self.device, stream):
                return self.evict(weights, lens, keep, first, recent, positions, status)
        dev = self._index
        a = VbKv8EvictArgs.from_buffer_copy(self._evict_args)
        a.weights = self._tracked(weights, "weights", torch.float32, None)
        a.room = room = weights.shape[2]
        if positions is not None:
            a.positions = self._tracked(positions, "positions", torch.int32, room)
        a.lens = _ints(lens, "lens", self.batch, dev)
        if not (0 < keep < 1 << 31 and 0 <= first and 0 <= recent and first + recent <= keep):
            raise ValueError(f"keep={keep} (1 to 2^31 - 1), first={first}, recent={recent}: neither "
                             "is negative, together they are at most keep")
        a.keep, a.first, a.recent = keep, first, recent
        if status is not None:
            a.status = status_ptr(status, dev)
        need = self._need.get(("evict", room, keep))
        if need is None:
            need = self._need["evict", room, keep] = lib.vb_kv8_evict_workspace_size(C.byref(a))
        st = current_stream(dev)
        if need:
            ws = _lists.get(need, self.device, st)
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
        after = torch.empty_like(lens)
        a.lens_out = after.data_ptr()
        check(lib.vb_kv8_evict(C.byref(a), st), "vb_kv8_evict")
        return after


__all__ = ["PagedKV8Cache", "SharedPrefix"]

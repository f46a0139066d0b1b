"""Paged KV caches and packed rows: a cache in pages that a table names, so that
sequences of any lengths share a memory, and agents the pages of a common
prefix; and attention of whole packed prompts on their own rows.

Python view of pkv_paged_store / pkv_paged_load, pkv_paged_attend and pkv_prompts
(include/pkv_codec.h).  torch supplies memory and streams only; every call is
asynchronous and can be captured into a graph.  No gradients: a cache is served,
not trained.

Rows of several sequences are packed one sequence behind the other along one
axis.  The same words describe them to every call:
  tables  int32 [sequences, pages of a sequence]: slot j of sequence s is place
          j % page_size of page tables[s, j // page_size].  A number that is no
          page's names none: its slots are not stored to, loaded as 0 and seen
          by no row
  lens    int32 [sequences], or one int for all: slots of each sequence, the
          packed rows' own counted; its rows are its last slots
  starts  int32 [sequences + 1], ascending: the rows of sequence s are starts[s]
          .. starts[s + 1] - 1; None: as many for each (rows / sequences)
All are device tensors, read on the device, so that a captured call replays with
new ones.
"""
from __future__ import annotations

import ctypes as C
import math

from . import _lib as L
from .live import DeviceCalls, _fits, _like, _rows_dtype, _strides


def _pages_dtype(t):
    import torch
    return {torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16, torch.uint8: L.DT_FP8,
            torch.float8_e4m3fn: L.DT_FP8}.get(t)


def _starts(starts, seqs: int, dev):
    import torch
    if starts.dtype != torch.int32 or starts.shape != (seqs + 1,) or not starts.is_contiguous() or starts.device != dev:
        raise ValueError(f"starts must be a contiguous int32 tensor of {seqs + 1} on the device of the call")
    return starts


def _whole(t) -> bool:
    """Strides and address that the kernels read, channels in line."""
    unit = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in _strides(t)[:-1])


class PagedKVCache(DeviceCalls):
    """A KV cache in pages of `page_size` slots (a power of two, 16 to 65,536):
    buf [layers, pages, K|V, heads, page_size, dim], bfloat16 or float16, or in
    8 bits a value (torch.float8_e4m3fn or uint8: OCP MX FP8, e4m3 codes with one
    power-of-two scale byte per 32 values along head_dim; 8.25 bits in all) with
    scales uint8 [.., dim / 32].  One table serves all layers.  ``store`` rounds
    rows into the slots of their sequences, ``load`` gives the values they hold,
    ``attend`` works on the pages themselves.  Who gets which page is the
    caller's."""

    def __init__(self, layers: int, heads: int, pages: int, page_size: int, dim: int, dtype=None, device="cuda"):
        import torch
        shape = (layers, pages, 2, heads, page_size, dim)
        buf = torch.zeros(shape, dtype=torch.uint8 if _pages_dtype(dtype) == L.DT_FP8 else dtype or torch.bfloat16,
                          device=device)
        scales = None
        if buf.dtype == torch.uint8:
            scales = torch.zeros((*shape[:5], dim // 32), dtype=torch.uint8, device=device)
        self._set(buf, scales)

    @classmethod
    def over(cls, buf, scales=None) -> "PagedKVCache":
        """A cache over a caller's tensors (contiguous; kept, not copied)."""
        self = cls.__new__(cls)
        self._set(buf, scales)
        return self

    def _set(self, buf, scales):
        import torch
        if _pages_dtype(buf.dtype) is None:
            raise TypeError("pages are bfloat16, float16 or 8 bits (float8_e4m3fn or uint8)")
        if buf.dim() != 6 or buf.shape[2] != 2 or not buf.is_contiguous():
            raise ValueError("buf must be a contiguous [layers, pages, 2, heads, page_size, dim] tensor")
        self.layers, self.pages, _, self.heads, self.page_size, self.dim = buf.shape
        if self.dim not in (64, 128):
            raise ValueError("head_dim 64 or 128")
        if not 16 <= self.page_size <= 65536 or self.page_size & (self.page_size - 1):
            raise ValueError("page_size is a power of two, 16 to 65536")
        if (scales is not None) != (_pages_dtype(buf.dtype) == L.DT_FP8):
            raise ValueError("8-bit pages, and only they, have scales")
        if scales is not None and (scales.dtype != torch.uint8 or scales.shape != (*buf.shape[:5], self.dim // 32) or
                                   not scales.is_contiguous() or scales.device != buf.device):
            raise ValueError("scales must be a contiguous uint8 [layers, pages, 2, heads, page_size, dim / 32]")
        self.buf, self.scales = buf, scales

    @property
    def device(self):
        return self.buf.device

    # ------------------------------------------------------------ the call's words
    def _view(self, layer=None) -> "L.PageView":
        """The cache, or one layer of it, but for the addresses."""
        side = self.heads * self.page_size * self.dim
        if layer is not None and not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} outside the cache")
        elems = self.buf.numel() - side - (layer or 0) * 2 * self.pages * side
        return L.PageView(None, None, None, None, 2 * self.pages * side, 2 * side, self.page_size * self.dim, self.dim,
                          elems, self.layers if layer is None else 1, self.pages, self.heads, self.page_size, self.dim,
                          _pages_dtype(self.buf.dtype))

    def _point(self, view, layer) -> None:
        """The addresses of a view, as the cache's memory is now."""
        side, size = self.heads * self.page_size * self.dim, self.buf.element_size()
        first = (layer or 0) * 2 * self.pages * side
        p = self.buf.data_ptr()
        view.d_keys, view.d_values = p + first * size, p + (first + side) * size
        if self.scales is not None:
            p = self.scales.data_ptr()
            view.d_key_scales, view.d_value_scales = p + first // 32, p + (first + side) // 32

    def _memory(self):
        """What a kept struct depends on in the cache's memory besides its address."""
        return self.buf.numel(), self.buf.dtype, None if self.scales is None else self.scales.numel()

    def _tables(self, tables):
        import torch
        if tables.dim() != 2 or tables.dtype != torch.int32 or not tables.shape[0] or not tables.shape[1] or \
                (tables.shape[1] > 1 and tables.stride(1) != 1):
            raise ValueError("tables must be an int32 [sequences, pages of a sequence], a sequence's in line")
        return tables

    def _sequences(self, tables, rows: int, starts) -> "L.Sequences":
        """The struct of a call's words but for the addresses."""
        seqs = tables.shape[0]
        if starts is None and rows % seqs:
            raise ValueError(f"{rows} rows are not as many for each of {seqs} sequences: give their starts")
        return L.Sequences(None, _strides(tables)[0], None, None, seqs, tables.shape[1], rows, 0)

    def _words(self, seqs, tables, lens, starts):
        """Addresses of the words; what they belong to must outlive the launch."""
        import torch
        n = tables.shape[0]
        if not isinstance(lens, torch.Tensor):
            lens = torch.full((n,), int(lens), dtype=torch.int32, device=self.device)
        if lens.dtype != torch.int32 or lens.shape != (n,) or not lens.is_contiguous() or lens.device != self.device:
            raise ValueError(f"lens must be a contiguous int32 tensor of {n} on the cache's device")
        seqs.d_tables, seqs.d_lens = tables.data_ptr(), lens.data_ptr()
        seqs.d_starts = None if starts is None else _starts(starts, n, self.device).data_ptr()
        return lens

    # ------------------------------------------------------------ rows in and out
    def _rows(self, entry, keys, values, tables, lens, starts, layer, handle, ctx):
        """One store or load of tensors that fit."""
        some = keys if keys is not None else values

        def make():
            s = _strides(some)
            s = s if layer is None else [0, *s]
            return L.PagedRowsOp(self._view(layer), self._sequences(tables, some.shape[-3], starts), None, None,
                                 s[0], s[1], s[2], _rows_dtype(some.dtype), 0), None

        op, _ = self._plan((0, layer, self._memory(), _like(some), _like(tables), starts is None), make)
        self._point(op.pages, layer)
        lens = self._words(op.seqs, tables, lens, starts)
        if keys is not None:
            op.d_keys = keys.data_ptr()
        if values is not None:
            op.d_values = values.data_ptr()
        L.check(getattr(L.lib(), entry)(ctx.ptr, C.byref(op), handle), entry)

    def store(self, keys, values, tables, lens, starts=None, layer: int | None = None, stream=None) -> None:
        """Put packed rows [layers, rows, heads, dim] of float32, bfloat16 or
        float16 keys and values (None: that side is left alone) into their
        sequences' last slots, of every layer, or without the layers axis into one
        layer's.  Rounded to nearest even; 8-bit pages: each block of 32 values
        takes the smallest power-of-two scale that keeps the largest within 448
        steps, each value its nearest code; a block with an infinity or NaN
        becomes NaN.  A row whose slot is negative or has no page is not stored.
        Two rows must not have the same place of the same page: sequences that
        share pages store into pages of their own.  Rows that lie among the
        pages themselves are refused (load them first), as are rows or pages that
        carry a gradient or a tangent."""
        some = keys if keys is not None else values
        if some is None:
            return
        for t in (keys, values):
            if t is None:
                continue
            if _rows_dtype(t.dtype) is None or t.dtype != some.dtype:
                raise TypeError("keys and values are both float32, bfloat16 or float16")
            lead = 1 if layer is None else 0
            if t.dim() != 3 + lead or t.shape != some.shape or t.shape[lead + 1:] != (self.heads, self.dim) or \
                    (lead and t.shape[0] != self.layers):
                raise ValueError(f"keys and values must be [{'layers, ' if lead else ''}rows, {self.heads}, {self.dim}]")
        self._served(keys, "store", values, self.buf)
        dev = self.device
        self._tables(tables)
        self._on_device(dev, keys, values, tables)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            if not _whole(some) or (values is not None and values is not some and
                                    (values.stride() != some.stride() or values.data_ptr() % 16)):
                keys, values = (None if t is None else t.contiguous() for t in (keys, values))
                keys, values = (t if t is None or t.data_ptr() % 16 == 0 else t.clone() for t in (keys, values))
            self._rows("pkv_paged_store", keys, values, tables, lens, starts, layer, handle, ctx)

    def load(self, rows: int, tables, lens, starts=None, layer: int | None = None, dtype=None, stream=None):
        """What the last slots of the sequences hold, `rows` in all: (keys,
        values), packed [layers, rows, heads, dim] (no layers axis for one layer)
        of dtype (bfloat16 unless given; exact in float32, and in bfloat16 from 8
        bits).  Whole sequences: starts the running sum of lens.  Rows whose slot
        is negative or has no page, or that are no sequence's, are 0.  Pages that
        carry a gradient or a tangent are refused."""
        import torch
        dtype = dtype or torch.bfloat16
        if _rows_dtype(dtype) is None:
            raise TypeError("load gives float32, bfloat16 or float16")
        if rows < 0:
            raise ValueError("rows is not negative")
        self._served(self.buf, "load")
        dev = self.device
        self._tables(tables)
        self._on_device(dev, tables)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            shape = (rows, self.heads, self.dim) if layer is not None else (self.layers, rows, self.heads, self.dim)
            keys, values = (torch.empty(shape, dtype=dtype, device=dev) for _ in range(2))
            self._rows("pkv_paged_load", keys, values, tables, lens, starts, layer, handle, ctx)
        return keys, values

    # ------------------------------------------------------------ attention
    def attend(self, layer: int, q, tables, lens, starts=None, window: int = 0, sinks: int = 0,
               scale: float | None = None, lse=None, out=None, max_rows: int | None = None, max_len: int | None = None,
               stream=None):
        """Attention of packed query rows q [rows, query heads, dim] over one
        layer: single tokens, chunks of prompts, or both.  A row sees the slots of
        its sequence up to its own -- all of them, or with window > 0 the last
        `window` and the first `sinks`.  Query heads are a multiple of the cache's
        heads, neighbours sharing one.  A row that sees nothing gives 0.  scale: 1
        / sqrt(dim) unless given.

        q has the pages' dtype; over 8-bit pages bfloat16 or float16.  Returns out
        (q's shape and dtype); rows that are no sequence's are left alone in an
        `out` that is given, and 0 in a new one.  lse: float32 [query heads,
        rows], the rows' log of the sum of exponentials.  max_rows, max_len: no
        sequence has more rows or slots (an int `lens` says so itself); they size
        the launch.  Of a sequence that has more rows, those past max_rows are no
        sequence's; a length past max_len is taken as max_len.

        Tensors that carry a gradient or a tangent, the pages among them, are
        refused: there is no derivative."""
        import torch
        dev = self.device
        self._tables(tables)
        self._on_device(dev, q, tables, lse, out)
        self._served(q, "attend", self.buf, lse, out)
        sized = None      # by an int length: the call's own, so that a loop over lengths keeps one struct
        if max_len is None and not isinstance(lens, torch.Tensor):
            sized = min(max(int(lens), 1), tables.shape[1] * self.page_size)

        def plan(q):
            return self._plan((1, layer, self._memory(), _like(q), _like(tables), starts is None, window, sinks, scale,
                               max_rows, max_len, _like(lse), _like(out)),
                              lambda: self._attend_op(layer, q, tables, starts, window, sinks, scale, lse, out, max_rows,
                                                      max_len))

        op, (need, fits) = plan(q)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            if not fits or q.data_ptr() % 16:
                q = q.clone(memory_format=torch.contiguous_format)
                op, (need, _) = plan(q)
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=dev)
                op.clear = 0 if starts is None else 1
            self._point(op.pages, layer)
            lens = self._words(op.seqs, tables, lens, starts)
            op.d_q, op.d_out = q.data_ptr(), out.data_ptr()
            if lse is not None:
                op.d_lse = lse.data_ptr()
            if sized is not None:
                op.max_len = sized
                need = op.workspace_bytes = L.lib().pkv_paged_attend_workspace(C.byref(op))
            if need:
                work = torch.empty(need, dtype=torch.uint8, device=dev)
                op.d_workspace = work.data_ptr()
            rc = L.lib().pkv_paged_attend(ctx.ptr, C.byref(op), handle)
            if rc:
                L.check(rc, "pkv_paged_attend")
        return out

    def _attend_op(self, layer, q, tables, starts, window, sinks, scale, lse, out, max_rows, max_len):
        """The call's struct but for the addresses, its workspace bytes, and
        whether q's strides are the kernels' (if not, the call copies it)."""
        import torch
        if q.dtype not in (torch.bfloat16, torch.float16) or (self.scales is None and self.buf.dtype != q.dtype):
            raise TypeError("q must have the pages' dtype (bfloat16 or float16 over 8-bit pages)")
        if q.dim() != 3 or q.shape[2] != self.dim or not q.shape[1] or q.shape[1] % self.heads:
            raise ValueError(f"q must be [rows, a multiple of {self.heads} query heads, {self.dim}]")
        words = self._sequences(tables, q.shape[0], starts)
        if max_len is not None and not 1 <= max_len <= tables.shape[1] * self.page_size:
            raise ValueError(f"max_len is 1 .. {tables.shape[1] * self.page_size}")
        s = _shape(q, window, sinks, scale, lse, out, max_rows, self.dim)
        op = L.PagedAttendOp(self._view(layer), words, None, None, s.q[0], s.q[1], s.out[0], s.out[1], None, None, 0, s.scale,
                             s.dtype, q.shape[1], max_rows or 0, max_len or 0, s.window, s.sinks, 0)
        # whether there are starts is all of their address that a workspace's size goes by
        op.seqs.d_starts = None if starts is None else 16
        op.workspace_bytes = L.lib().pkv_paged_attend_workspace(C.byref(op))
        return op, (op.workspace_bytes, s.fits)


class _shape:
    """What both attention calls check of q, out and lse, and their strides."""

    def __init__(self, q, window, sinks, scale, lse, out, max_rows, dim):
        import torch
        rows, heads = q.shape[0], q.shape[1]
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks are not negative")
        if max_rows is not None and max_rows < 1:
            raise ValueError("max_rows is at least 1")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not _fits(out)):
            raise ValueError("out must have q's shape and dtype, rows of 16-byte pieces")
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != (heads, rows) or not lse.is_contiguous()):
            raise ValueError(f"lse must be a contiguous float32 [{heads}, {rows}]")
        self.q = _strides(q)
        self.out = _strides(out) if out is not None else [heads * dim, dim]     # a new out is contiguous
        self.scale = 1.0 / math.sqrt(dim) if scale is None else scale
        self.dtype = _rows_dtype(q.dtype)
        self.window, self.sinks = min(window, 0xffffffff), min(sinks, 0xffffffff)
        self.fits = _fits_rows(q)


def _fits_rows(t) -> bool:
    return t.stride(2) == 1 and all(s % 8 == 0 for s in _strides(t)[:2])


class _Prompts(DeviceCalls):
    _what = "q"

    def __call__(self, q, k, v, starts, window, sinks, scale, lse, out, max_rows, stream):
        import torch
        dev = q.device
        self._on_device(dev, k, v, starts, lse, out)
        self._served(q, "attend_prompts", k, v, lse, out)

        def plan(q, k, v):
            return self._plan((_like(q), _like(k), _like(v), starts.shape, window, sinks, scale, _like(lse), _like(out),
                               max_rows), lambda: self._op(q, k, v, starts, window, sinks, scale, lse, out, max_rows))

        op, (need, fits) = plan(q, k, v)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            if not fits or (q.data_ptr() | k.data_ptr() | v.data_ptr()) % 16:
                q, k, v = (t if _whole(t) else t.clone(memory_format=torch.contiguous_format) for t in (q, k, v))
                op, (need, _) = plan(q, k, v)
            if out is None:
                out = torch.empty(q.shape, dtype=q.dtype, device=dev)
                op.clear = 1
            op.d_q, op.d_k, op.d_v, op.d_out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
            op.d_starts = _starts(starts, starts.shape[0] - 1, dev).data_ptr()
            if lse is not None:
                op.d_lse = lse.data_ptr()
            if need:
                work = torch.empty(need, dtype=torch.uint8, device=dev)
                op.d_workspace = work.data_ptr()
            rc = L.lib().pkv_prompts(ctx.ptr, C.byref(op), handle)
            if rc:
                L.check(rc, "pkv_prompts")
        return out

    def _op(self, q, k, v, starts, window, sinks, scale, lse, out, max_rows):
        import torch
        if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError("q, k and v are all bfloat16 or float16")
        if q.dim() != 3 or q.shape[2] not in (64, 128):
            raise ValueError("q must be [rows, query heads, head_dim 64 or 128]")
        if k.dim() != 3 or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or not k.shape[1] or \
                not q.shape[1] or q.shape[1] % k.shape[1] or v.shape != k.shape:
            raise ValueError("k and v must be [rows, heads, head_dim] of q's rows, query heads a multiple of heads")
        if starts.dim() != 1 or starts.shape[0] < 2:
            raise ValueError("starts must be [sequences + 1]")
        s = _shape(q, window, sinks, scale, lse, out, max_rows, q.shape[2])
        ks, vs = _strides(k), _strides(v)
        op = L.PromptsOp(None, None, None, None, s.q[0], s.q[1], ks[0], ks[1], vs[0], vs[1], s.out[0], s.out[1], None, None,
                         None, 0, s.scale, s.dtype, starts.shape[0] - 1, q.shape[0], k.shape[1], q.shape[1], q.shape[2],
                         max_rows or 0, s.window, s.sinks, 0)
        op.workspace_bytes = L.lib().pkv_prompts_workspace(C.byref(op))
        return op, (op.workspace_bytes, s.fits and _fits_rows(k) and _fits_rows(v))


_prompts = _Prompts()


def attend_prompts(q, k, v, starts, window: int = 0, sinks: int = 0, scale: float | None = None, lse=None, out=None,
                   max_rows: int | None = None, stream=None):
    """Attention of whole packed prompts on their own rows: q [rows, query heads,
    dim], k and v [rows, heads, dim], all bfloat16 or float16, any strides with
    the channels in line (slices of one projection's output, for example).  Row i
    of a sequence sees that sequence's rows up to its own, or with window > 0 the
    last `window` and the first `sinks`.  Query heads are a multiple of heads,
    neighbours sharing one.  starts: int32 [sequences + 1].

    Returns out (q's shape and dtype); rows that are no sequence's are left alone
    in an `out` that is given, and 0 in a new one.  scale, lse, max_rows as
    ``PagedKVCache.attend``'s.  Tensors that carry a gradient or a tangent are
    refused: there is no derivative."""
    return _prompts(q, k, v, starts, window, sinks, scale, lse, out, max_rows, stream)

"""Live KV caches: attention over a cache, the cache held in 4 bits, and
eviction by accumulated attention weight.

Python view of pkv_attend, pkv_fp4_store / pkv_fp4_load and pkv_evict
(include/pkv_codec.h).  ``LiveCache`` gives a cache its ``attend`` and
``evict``; ``FourBitKVCache`` is the 4-bit sibling of ``pool.DeviceKVCache``.
torch supplies memory and streams only; every call is asynchronous and can be
captured into a graph.  No gradients: a cache is served, not trained.

Lengths, first slots and counts are int32 device tensors, one per cache copy
(so a captured graph replays with new ones), or one int for all copies.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math

import numpy as np

from . import _lib as L
from .device import device_context


_TYPES: dict = {}


def _rows_dtype(t):
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16})
    return _TYPES.get(t)


def _strides(t) -> list:
    """Strides with 0 where there is nothing to step over."""
    return [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]


def _fits(t) -> bool:
    """Rows of 16-byte pieces, as the kernels read and write them."""
    if t.is_contiguous() and t.shape[-1] % 8 == 0:
        return t.data_ptr() % 16 == 0
    unit = 16 // t.element_size()
    return t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(s % unit == 0 for s in _strides(t)[:-1])


def _like(t):
    """What a call's struct depends on in a tensor besides its address."""
    return None if t is None else (t.shape, t.dtype, t.stride())


_NO_GUARD = contextlib.nullcontext()


class DeviceCalls:
    """The frame of a call of the library: its device and stream, its kept
    struct, and what every call refuses.  _what: whose device it is."""

    _what = "the cache"

    def _frame(self, dev, stream):
        """(context, stream handle, guard): the guard makes the cache's device
        and the stream current, so that what a call allocates belongs to it."""
        import torch
        if dev.type != "cuda":
            raise ValueError(f"{self._what} is not on a GPU")
        index, now = dev.index, torch.cuda.current_device()
        if index is None:
            index = now
        if stream is not None:
            if stream.device_index != index:
                raise ValueError(f"the stream belongs to another device than {self._what}")
            return device_context(index), stream.cuda_stream, torch.cuda.stream(stream)
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # a Stream object costs as much as a launch
        handle = raw(index) if raw is not None else torch.cuda.current_stream(index).cuda_stream
        return device_context(index), handle, _NO_GUARD if index == now else torch.cuda.device(index)

    def _plan(self, key, make):
        """A copy of the call's struct for `key`, checked and filled once with
        what shapes, strides and types decide; every call sets its own
        addresses, those of the cache too."""
        plans = self.__dict__.setdefault("_plans", {})
        got = plans.get(key)
        if got is None:
            got = make()
            if len(plans) >= 256:
                plans.clear()
            plans[key] = got
        op, extra = got
        return type(op).from_buffer_copy(op), extra

    @staticmethod
    def _served(t, call: str, *more):
        """No gradient or tangent of a call's tensors is lost without a word."""
        import torch
        fwd = torch.autograd.forward_ad     # outside of any level nothing has a tangent
        level = getattr(fwd, "_current_level", 0) >= 0
        for x in (t, *more):
            if x is None:
                continue
            if x.requires_grad and torch.is_grad_enabled():
                raise ValueError(f"{call} has no backward pass: detach its tensors or call it under torch.no_grad()")
            if level and fwd.unpack_dual(x).tangent is not None:
                raise ValueError(f"{call} has no forward-mode derivative: give it the primal of a dual tensor")

    def _on_device(self, dev, *tensors):
        for t in tensors:
            if t is not None and t.device != dev:
                raise ValueError(f"a tensor is on {t.device}, {self._what} on {dev}")


class LiveCache(DeviceCalls):
    """What a cache of [copies][layers][K|V][heads][tokens][dim] rows does on
    the device.  A subclass has copies, layers, heads, tokens, dim, device and
    _pointers(): (dtype, bytes of an element or None for 4-bit codes, keys,
    values, key scales, value scales, elements of the whole memory)."""

    def _view(self, layer=None) -> "L.KvView":
        """The cache, or one layer of it."""
        memory = self._pointers()
        dtype, elems = memory[0], memory[6]
        side = self.heads * self.tokens * self.dim
        per_layer = 2 * side
        if layer is not None and not 0 <= layer < self.layers:
            raise IndexError(f"layer {layer} outside the cache")
        elems -= side + (layer or 0) * per_layer
        if elems < 0:
            raise ValueError("the cache's memory is smaller than its shape")
        view = L.KvView(None, None, None, None, self.layers * per_layer, per_layer, self.tokens * self.dim,
                        self.dim, elems, self.copies, 1 if layer is not None else self.layers, self.heads,
                        self.tokens, self.dim, dtype)
        self._point(view, layer, memory)
        return view

    def _point(self, view, layer, memory) -> None:
        """The addresses of a view, as the cache's memory is now."""
        _, size, k, v, ks, vs, _ = memory
        first = (layer or 0) * 2 * self.heads * self.tokens * self.dim
        if size is None:
            view.d_keys, view.d_values = k + first // 2, v + first // 2
            view.d_key_scales, view.d_value_scales = ks + first // 32, vs + first // 32
        else:
            view.d_keys, view.d_values = k + first * size, v + first * size

    def _words(self, x, name: str):
        """int32 device words, one per copy."""
        import torch
        if not isinstance(x, torch.Tensor):
            return torch.full((self.copies,), int(x), dtype=torch.int32, device=self.device)
        if x.dtype != torch.int32 or x.shape != (self.copies,) or not x.is_contiguous() or x.device != self.device:
            raise ValueError(f"{name} must be a contiguous int32 tensor of {self.copies} on the cache's device")
        return x

    # ------------------------------------------------------------ attention
    def attend(self, layer: int, q, lens, q_lens=None, window: int = 0, sinks: int = 0, scale: float | None = None,
               weights=None, lse=None, out=None, max_len: int | None = None, stream=None):
        """Attention of query rows q [copies, rows, query heads, dim] over one
        layer: row i of copy c stands at slot lens[c] - q_lens[c] + i (q_lens:
        all rows unless given; rows behind it are padding and left alone in
        `out`) and sees the slots up to its own -- all of them, or with
        window > 0 the last `window` and the first `sinks`.  Query heads are a
        multiple of the cache's heads, neighbours sharing one.  A row that
        sees nothing gives 0.  scale: 1 / sqrt(dim) unless given.

        q has the cache's dtype; over a FourBitKVCache any of float32,
        bfloat16 and float16.  Returns out (q's shape and dtype).
        weights: float32 [copies, heads, tokens] to which every slot's softmax
        weight, summed over the rows and the query heads of its head, is
        added.  lse: float32 [copies, query heads, rows], the rows' log of the
        sum of exponentials.  max_len: no length is above it (an int `lens`
        says so itself); sizes the launch.

        A q that carries a gradient or a tangent is refused: there is no
        derivative."""
        import torch
        dev = self.device
        self._on_device(dev, q, weights, lse, out)
        self._served(q, "attend")
        sized = None      # by an int length: the call's own, so that a loop over lengths keeps one struct
        if max_len is None:
            max_len = self.tokens
            if not isinstance(lens, torch.Tensor):
                sized = min(max(int(lens), 1), self.tokens)

        memory = self._pointers()

        def plan(q):
            return self._plan((0, layer, _like(q), window, sinks, scale, max_len, memory[0], memory[6], _like(weights),
                               _like(lse), _like(out)),
                              lambda: self._attend_op(layer, q, window, sinks, scale, weights, lse, out, max_len))

        op, (need, fits) = plan(q)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            if not fits or q.data_ptr() % 16:
                q = q.clone(memory_format=torch.contiguous_format)
                op, (need, _) = plan(q)
            lens = self._words(lens, "lens")
            op.d_lens = lens.data_ptr()
            if out is None:
                # rows behind q_lens are nobody's: 0 rather than whatever the memory held
                out = (torch.empty if q_lens is None else torch.zeros)(q.shape, dtype=q.dtype, device=dev)
            self._point(op.cache, layer, memory)
            op.d_q, op.d_out = q.data_ptr(), out.data_ptr()
            if q_lens is not None:
                q_lens = self._words(q_lens, "q_lens")
                op.d_q_lens = q_lens.data_ptr()
            if weights is not None:
                op.d_weights = weights.data_ptr()
            if lse is not None:
                op.d_lse = lse.data_ptr()
            if sized is not None:
                op.max_len = sized
                need = op.workspace_bytes = L.lib().pkv_attend_workspace(C.byref(op))
            if need:
                work = torch.empty(need, dtype=torch.uint8, device=dev)
                op.d_workspace = work.data_ptr()
            rc = L.lib().pkv_attend(ctx.ptr, C.byref(op), handle)
            if rc:
                L.check(rc, "pkv_attend")
        return out

    def _attend_op(self, layer, q, window, sinks, scale, weights, lse, out, max_len):
        """The call's struct but for the addresses, its workspace bytes, and
        whether q's strides are the kernels' (if not, the call copies it)."""
        import torch
        dtype = _rows_dtype(q.dtype)
        if dtype is None or (not isinstance(self, FourBitKVCache) and self.buf.dtype != q.dtype):
            raise TypeError("q must have the cache's dtype (float32, bfloat16 or float16 over a 4-bit cache)")
        if q.dim() != 4 or q.shape[0] != self.copies or q.shape[3] != self.dim:
            raise ValueError(f"q must be [{self.copies}, rows, query heads, {self.dim}]")
        rows, heads = q.shape[1], q.shape[2]
        if not heads or heads % self.heads:
            raise ValueError(f"{heads} query heads over {self.heads} heads")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks are not negative")
        if not 1 <= max_len <= self.tokens:
            raise ValueError(f"max_len is 1 .. {self.tokens}")
        if out is not None and (out.shape != q.shape or out.dtype != q.dtype or not _fits(out)):
            raise ValueError("out must have q's shape and dtype, rows of 16-byte pieces")
        # a new out is contiguous
        os = _strides(out) if out is not None else [rows * heads * self.dim, heads * self.dim, self.dim]
        qs = _strides(q)
        op = L.AttendOp(self._view(layer), None, None, qs[0], qs[1], qs[2], os[0], os[1], os[2], None, None, None, None, 0, 0, None, 0,
                        1.0 / math.sqrt(self.dim) if scale is None else scale, dtype, heads, rows, max_len,
                        min(window, 0xffffffff), min(sinks, 0xffffffff), 0)
        if weights is not None:
            if weights.dtype != torch.float32 or weights.shape != (self.copies, self.heads, self.tokens) or \
                    weights.stride(2) != 1:
                raise ValueError(f"weights must be float32 [{self.copies}, {self.heads}, {self.tokens}], "
                                 "slots contiguous")
            ws = _strides(weights)
            op.d_weights, op.weight_copy_stride, op.weight_head_stride = weights.data_ptr(), ws[0], ws[1]
        if lse is not None and (lse.dtype != torch.float32 or lse.shape != (self.copies, heads, rows) or
                                not lse.is_contiguous()):
            raise ValueError(f"lse must be a contiguous float32 [{self.copies}, {heads}, {rows}]")
        op.workspace_bytes = L.lib().pkv_attend_workspace(C.byref(op))
        unit = 16 // q.element_size()
        return op, (op.workspace_bytes, q.stride(3) == 1 and all(n % unit == 0 for n in qs[:3]))

    # ------------------------------------------------------------ eviction
    def evict(self, lens, weights, budget: int, sinks: int = 0, recent: int = 0, layer: int | None = None, into=None,
              stream=None):
        """Shorten every head of a layer (of all layers: layer=None) to at
        most `budget` slots: the first `sinks`, the last `recent` and the
        heaviest of the others by `weights` (float32 [copies, layers, heads,
        tokens], without the layers axis for one layer; ties to the lower
        slot) are kept and packed in their order to the front, in place or in
        `into` (a cache of the same kind, copies, layers, heads and dim, with
        room for the budget).

        Returns (kept, lens, weights): the kept slots int32 [copies, layers,
        heads, budget], -1 behind the last; the new lengths int32 [copies];
        the kept slots' weights, 0 behind them -- `weights` itself in place, a
        new tensor of `into`'s slots otherwise.  An all-layer call takes one
        length per copy for all layers."""
        import torch
        to, dev = self if into is None else into, self.device
        lead = (self.copies, self.layers, self.heads) if layer is None else (self.copies, self.heads)
        memory = self._pointers()
        room = memory if into is None else to._pointers()
        if to.device != dev:
            raise ValueError("into is on another device")
        self._on_device(dev, weights)

        def make():
            if room[0] != memory[0] or (to.copies, to.layers, to.heads, to.dim) != \
                    (self.copies, self.layers, self.heads, self.dim):
                raise ValueError("into must be a cache of the same kind, copies, layers, heads and dim")
            if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
                raise ValueError("the budget holds at least one slot, the sinks and the recent slots")
            if to.tokens < min(budget, self.tokens):
                raise ValueError(f"into has {to.tokens} slots, the budget is {budget}")
            if weights.dtype != torch.float32 or weights.shape != (*lead, self.tokens) or weights.stride(-1) != 1:
                raise ValueError(f"weights must be float32 {[*lead, self.tokens]}, slots contiguous")
            op = L.EvictOp(self._view(layer), to._view(layer))
            out = _strides(weights)
            if into is not None:   # contiguous
                out = [math.prod(lead[k + 1:]) * to.tokens for k in range(len(lead))]
            for dst, s in ((op.weight_strides, _strides(weights)), (op.out_strides, out)):
                dst[:] = s[:3] if layer is None else (s[0], 0, s[1])
            op.budget, op.sinks, op.recent = budget, sinks, recent
            return op, None

        key = (1, layer, budget, sinks, recent, memory[0], memory[6], _like(weights),
               None if into is None else (room[0], room[6], to.copies, to.layers, to.heads, to.tokens, to.dim))
        op, _ = self._plan(key, make)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            lens = self._words(lens, "lens")
            new_lens = torch.empty_like(lens)
            kept = torch.empty((*lead, budget), dtype=torch.int32, device=dev)
            packed = weights if into is None else torch.empty((*lead, to.tokens), dtype=torch.float32, device=dev)
            self._point(op.cache, layer, memory)
            to._point(op.into, layer, room)
            op.d_lens, op.d_new_lens, op.d_kept = lens.data_ptr(), new_lens.data_ptr(), kept.data_ptr()
            op.d_weights, op.d_weights_out = weights.data_ptr(), packed.data_ptr()
            L.check(L.lib().pkv_evict(ctx.ptr, C.byref(op), handle), "pkv_evict")
        if layer is None:
            filled = min(self._seq_len, budget)
            to._seq_len = filled if to is self else max(to._seq_len, filled)
        return kept, new_lens, packed


class FourBitKVCache(LiveCache):
    """A KV cache of the layout of ``pool.DeviceKVCache`` held in 4 bits a value
    (OCP MX FP4: e2m1 codes, one power-of-two scale byte per 32 values along
    head_dim; 4.25 bits in all): codes uint8 [copies, layers, 2, heads, tokens,
    dim / 2], scales uint8 [.., dim / 32].  ``store`` rounds rows into slots,
    ``load`` gives the values they stand for, ``attend`` and ``evict`` work on
    the codes themselves.  Also proveKV's ``CacheTarget``
    (proveKV/src/pool.rs:646-658), as DeviceKVCache."""

    def __init__(self, layers: int, heads: int, tokens: int, dim: int, copies: int = 1, device="cuda"):
        import torch
        if dim not in (64, 128):
            raise ValueError("head_dim 64 or 128")
        self.layers, self.heads, self.tokens, self.dim, self.copies = layers, heads, tokens, dim, copies
        shape = (copies, layers, 2, heads, tokens)
        self.codes = torch.zeros((*shape, dim // 2), dtype=torch.uint8, device=device)
        self.scales = torch.zeros((*shape, dim // 32), dtype=torch.uint8, device=device)
        self._seq_len = 0

    @classmethod
    def over(cls, codes, scales) -> "FourBitKVCache":
        """A cache over a caller's tensors (contiguous; kept, not copied)."""
        import torch
        if codes.dim() != 6 or codes.shape[2] != 2 or codes.shape[5] not in (32, 64) or \
                scales.shape != (*codes.shape[:5], codes.shape[5] // 16) or codes.device != scales.device:
            raise ValueError("codes [copies, layers, 2, heads, tokens, dim / 2], scales [.., dim / 32]")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or \
                not (codes.is_contiguous() and scales.is_contiguous()):
            raise ValueError("codes and scales must be contiguous uint8 tensors")
        self = cls.__new__(cls)
        self.copies, self.layers, _, self.heads, self.tokens, half = codes.shape
        self.dim = 2 * half
        self.codes, self.scales = codes, scales
        self._seq_len = 0
        return self

    @property
    def device(self):
        return self.codes.device

    def _pointers(self):
        side = self.heads * self.tokens * self.dim
        c, s = self.codes.data_ptr(), self.scales.data_ptr()
        return L.DT_FP4, None, c, c + side // 2, s, s + side // 32, min(2 * self.codes.numel(), 32 * self.scales.numel())

    # ------------------------------------------------------------ rows in and out
    def _rows(self, entry, keys, values, first, counts, layer, dev, stream_frame):
        """One store or load of tensors that fit; returns what must outlive the launch."""
        some = keys if keys is not None else values

        def make():
            ks = _strides(some)
            ks = ks if layer is None else [ks[0], 0, *ks[1:]]
            return L.RowsOp(self._view(layer), None, None, ks[0], ks[1], ks[2], ks[3], None, None,
                            _rows_dtype(some.dtype), some.shape[-2]), None

        memory = self._pointers()
        op, _ = self._plan((2, layer, memory[6], _like(some)), make)
        self._point(op.cache, layer, memory)
        ctx, handle = stream_frame
        first = self._words(first, "first")
        op.d_first = first.data_ptr()
        if counts is not None:
            counts = self._words(counts, "counts")
            op.d_counts = counts.data_ptr()
        if keys is not None:
            op.d_keys = keys.data_ptr()
        if values is not None:
            op.d_values = values.data_ptr()
        L.check(getattr(L.lib(), entry)(ctx.ptr, C.byref(op), handle), entry)

    def store(self, keys, values, first, layer: int | None = None, counts=None, stream=None) -> None:
        """Put rows [copies, layers, heads, rows, dim] of float32, bfloat16 or
        float16 keys and values (None: that side is left alone) into the slots
        first[c], first[c] + 1, .. of every layer, or without the layers axis
        into one layer's.  counts: rows of each copy (the others are padding).
        A row whose slot is outside the cache is not stored.  Each block of 32
        values takes the smallest power-of-two scale that keeps the largest
        within 7 steps, each value its nearest code; a block with an infinity
        or NaN becomes NaN.  Rows that carry a gradient or a tangent are
        refused, as by `attend`."""
        lead = (self.copies, self.layers, self.heads) if layer is None else (self.copies, self.heads)
        some = keys if keys is not None else values
        if some is None:
            return
        for t in (keys, values):
            if t is None:
                continue
            if _rows_dtype(t.dtype) is None or t.dtype != some.dtype:
                raise TypeError("keys and values are both float32, bfloat16 or float16")
            if t.shape != (*lead, some.shape[-2], self.dim):
                raise ValueError(f"keys and values must be {[*lead, 'rows', self.dim]}")
            self._served(t, "store")
        dev = self.device
        self._on_device(dev, keys, values)
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            if not _fits(some) or (values is not None and values is not some and
                                   (values.stride() != some.stride() or values.data_ptr() % 16)):
                keys, values = (None if t is None else t.contiguous() for t in (keys, values))
                keys, values = (t if t is None or t.data_ptr() % 16 == 0 else t.clone() for t in (keys, values))
            self._rows("pkv_fp4_store", keys, values, first, counts, layer, dev, (ctx, handle))

    def load(self, first, rows: int, layer: int | None = None, dtype=None, counts=None, stream=None):
        """The values that the slots first[c] .. first[c] + rows - 1 stand for:
        (keys, values), [copies, layers, heads, rows, dim] (no layers axis for
        one layer) of dtype (bfloat16 unless given; exact in bfloat16 and
        float32).  Rows without a slot, or behind counts[c], are 0."""
        import torch
        dtype = dtype or torch.bfloat16
        if _rows_dtype(dtype) is None:
            raise TypeError("load gives float32, bfloat16 or float16")
        if rows < 0:
            raise ValueError("rows is not negative")
        lead = (self.copies, self.layers, self.heads) if layer is None else (self.copies, self.heads)
        dev = self.device
        ctx, handle, guard = self._frame(dev, stream)
        with guard:
            keys, values = (torch.empty((*lead, rows, self.dim), dtype=dtype, device=dev) for _ in range(2))
            self._rows("pkv_fp4_load", keys, values, first, counts, layer, dev, (ctx, handle))
        return keys, values

    # ------------------------------------------------------------ CacheTarget
    def num_layers(self) -> int:
        return self.layers

    def _append(self, side: int, layer: int, position: int, vec) -> None:
        import torch
        if not (0 <= layer < self.layers and 0 <= position < self.tokens):
            raise IndexError(f"layer {layer} / position {position} outside the cache")
        v = torch.as_tensor(np.asarray(vec, dtype=np.float32)).reshape(1, self.heads, 1, self.dim).to(self.device)
        v = v.expand(self.copies, -1, -1, -1)
        self.store(v if side == 0 else None, v if side == 1 else None, position, layer=layer)
        self._seq_len = max(self._seq_len, position + 1)

    def append_key(self, layer: int, position: int, key) -> None:
        self._append(0, layer, position, key)

    def append_value(self, layer: int, position: int, value) -> None:
        self._append(1, layer, position, value)

    def seq_len(self) -> int:
        return self._seq_len

    def mark_filled(self, tokens: int) -> None:
        self._seq_len = max(self._seq_len, tokens)

"""Cache views of other strides than the caches of provekv_amd.pool, through the
C entries: heads inside slots, gaps between rows, keys and values interleaved."""
import ctypes as C

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [F32, BF16, F16, "fp4"]
IDS = ["f32", "bf16", "f16", "fp4"]
COPIES, HEADS = 3, 2


class Strided:
    """Rows [copies][slots][heads + 1][K|V][gap + dim], in codes and scales or
    elements; `rows` are the tensors of a [copies, heads, slots, ..] side."""

    def __init__(self, kind, T, D, fill):
        from provekv_amd import _lib as L
        fp4 = kind == "fp4"
        gap = D if fp4 else 16 // torch.empty(0, dtype=kind).element_size()
        unit = gap + D
        shape = (COPIES, T, HEADS + 1, 2)
        if fp4:
            self.parts = [torch.full((*shape, unit // 2), fill, dtype=torch.uint8, device="cuda"),
                          torch.full((*shape, unit // 32), fill, dtype=torch.uint8, device="cuda")]
            widths = D // 2, D // 32
        else:
            self.parts = [torch.full((*shape, unit), float(fill), dtype=kind, device="cuda")]
            widths = (D,)
        self.rows = [[p[:, :, :HEADS, side, -w:].permute(0, 2, 1, 3) for p, w in zip(self.parts, widths)]
                     for side in (0, 1)]
        slot = (HEADS + 1) * 2 * unit
        ptr = [[r.data_ptr() for r in side] for side in self.rows]
        elems = COPIES * T * slot - unit - gap
        self.view = L.KvView(ptr[0][0], ptr[1][0], ptr[0][1] if fp4 else None, ptr[1][1] if fp4 else None, T * slot, 0,
                             2 * unit, slot, elems, COPIES, 1, HEADS, T, D,
                             L.DT_FP4 if fp4 else {F32: L.DT_F32, BF16: L.DT_BF16, F16: L.DT_F16}[kind])

    def set(self, cache):
        for side in (0, 1):
            for r, p in zip(self.rows[side], parts(cache)):
                r.copy_(p[:, 0, side])
        return self


def parts(cache):
    return [cache.codes, cache.scales] if hasattr(cache, "codes") else [cache.buf]


def contiguous(kind, T, D, seed):
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    x = torch.randn(COPIES, 1, 2, HEADS, T, D, generator=torch.Generator().manual_seed(seed)).cuda()
    if kind != "fp4":
        return DeviceKVCache.over(x.to(kind))
    cache = FourBitKVCache(1, HEADS, T, D, copies=COPIES)
    cache.store(x[:, :, 0], x[:, :, 1], 0)
    return cache


def stream():
    return torch.cuda.current_stream().cuda_stream


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,T,window", [(1, 200, 0), (3, 131, 40), (50, 333, 0), (200, 300, 64)])
def test_attend(ctx, n, T, window, D, kind):
    """The bits of the same rows in a cache; gaps hold NaN patterns."""
    from provekv_amd import _lib as L
    cache = contiguous(kind, T, D, 1)
    other = Strided(kind, T, D, 255 if kind == "fp4" else float("nan")).set(cache)
    qt = BF16 if kind == "fp4" else kind
    G = 2
    q = torch.randn(COPIES, n, HEADS * G, D, generator=torch.Generator().manual_seed(2)).to(qt).cuda()
    lens = torch.tensor([T, T // 2, 7], dtype=torch.int32, device="cuda")
    w, lse = torch.zeros(COPIES, HEADS, T, device="cuda"), torch.zeros(COPIES, HEADS * G, n, device="cuda")
    want = cache.attend(0, q, lens, window=window, sinks=3, weights=w, lse=lse)
    out, w2, lse2 = torch.zeros_like(q), torch.zeros_like(w), torch.zeros_like(lse)
    rows = n * HEADS * G * D
    op = L.AttendOp(other.view, q.data_ptr(), out.data_ptr(), rows, HEADS * G * D, D, rows, HEADS * G * D, D,
                    lens.data_ptr(), None, lse2.data_ptr(), w2.data_ptr(), HEADS * T, T, None, 0, D ** -0.5,
                    {F32: L.DT_F32, BF16: L.DT_BF16, F16: L.DT_F16}[qt], HEADS * G, n, T, window, 3, 0)
    need = L.lib().pkv_attend_workspace(C.byref(op))
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    op.d_workspace, op.workspace_bytes = work.data_ptr(), need
    assert L.lib().pkv_attend(ctx.ptr, C.byref(op), stream()) == 0
    assert R.same(out, want) and R.same(w2, w) and R.same(lse2, lse)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
def test_store_load(ctx, D, dtype):
    from provekv_amd import _lib as L
    T, n = 50, 21
    other, cache = Strided("fp4", T, D, 17), contiguous("fp4", T, D, 3)
    other.set(cache)
    before = [p.clone() for p in other.parts]
    x = torch.randn(2, COPIES, 1, HEADS, n, D, generator=torch.Generator().manual_seed(4)).to(dtype).cuda()
    first = torch.tensor([0, 11, 40], dtype=torch.int32, device="cuda")
    cache.store(x[0], x[1], first)
    op = L.RowsOp(other.view, x[0].data_ptr(), x[1].data_ptr(), HEADS * n * D, 0, n * D, D, first.data_ptr(), None,
                  {F32: L.DT_F32, BF16: L.DT_BF16, F16: L.DT_F16}[dtype], n)
    assert L.lib().pkv_fp4_store(ctx.ptr, C.byref(op), stream()) == 0
    for side in (0, 1):
        for r, p, b in zip(other.rows[side], parts(cache), before):
            assert torch.equal(r, p[:, 0, side])
            r.copy_(torch.as_strided(b, r.shape, r.stride(), r.storage_offset()))
    for p, b in zip(other.parts, before):      # nothing but those rows was written
        assert torch.equal(p, b)
    other.set(cache)
    got = torch.full_like(x, 9.0)
    op.d_keys, op.d_values = got[0].data_ptr(), got[1].data_ptr()
    assert L.lib().pkv_fp4_load(ctx.ptr, C.byref(op), stream()) == 0
    for a, b in zip(got, cache.load(first, n, dtype=dtype)):
        assert R.same(a, b)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
def test_evict(ctx, in_place, D, kind):
    from provekv_amd import _lib as L
    T, budget = 900, 333
    cache = contiguous(kind, T, D, 5)
    other = Strided(kind, T, D, 3).set(cache)
    target = other if in_place else Strided(kind, budget + 2, D, 5)
    before = [p.clone() for p in target.parts]
    w = torch.rand(COPIES, 1, HEADS, T, generator=torch.Generator().manual_seed(6)).cuda()
    w2 = w.clone()
    lens = torch.tensor([T, 500, 100], dtype=torch.int32, device="cuda")
    kept, new, packed = cache.evict(lens, w, budget, sinks=2, recent=9)
    kept2, new2 = torch.zeros_like(kept), torch.zeros_like(new)
    slots = T if in_place else budget + 2
    out = w2 if in_place else torch.zeros(COPIES, 1, HEADS, slots, device="cuda")
    op = L.EvictOp(other.view, target.view, lens.data_ptr(), new2.data_ptr(), kept2.data_ptr(), w2.data_ptr(),
                   out.data_ptr(), (C.c_uint64 * 3)(HEADS * T, 0, T), (C.c_uint64 * 3)(HEADS * slots, 0, slots), budget, 2, 9, 0)
    assert L.lib().pkv_evict(ctx.ptr, C.byref(op), stream()) == 0
    assert torch.equal(kept2, kept) and torch.equal(new2, new) and torch.equal(out[..., :budget], packed[..., :budget])
    assert not out[..., budget:].any()
    for c, n in enumerate(new.tolist()):
        for side in (0, 1):
            for r, p, b in zip(target.rows[side], parts(cache), before):
                assert R.same(r[c, :, :n], p[c, 0, side, :, :n])
                r[c, :, :n] = torch.as_strided(b, r.shape, r.stride(), r.storage_offset())[c, :, :n]
    for p, b in zip(target.parts, before):     # nothing behind the kept rows, beside them or between them was written
        assert R.same(p, b)

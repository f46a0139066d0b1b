"""The paged-cache and packed-prompt calls' argument checks, on the CPU: the C
entries with the HIP runtime replaced by tests/host_live_hip.cpp (no pointer is
followed there), and the Python methods on memory of the host."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from test_live_host import CAPACITY, INVALID, OK, UNSUPPORTED, each, stub  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))
K, V, KS, VS, Q, OUT, TABLES, LENS, STARTS, WORK, LSE = (0x40000000 * (i + 1) for i in range(11))


@pytest.mark.parametrize("name", ["attend", "rows", "prompts", "sizes"])
def test_refusals(stub, name):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, name], capture_output=True, text=True,
                       timeout=120, env={**os.environ, "PYTHONPATH": os.pathsep.join((os.path.dirname(HERE), HERE))})
    assert r.returncode == 0, r.stdout + r.stderr


def view(L, dtype=1, layers=1, pages=10, H=2, P=32, D=64):
    # keys and values of [layers][pages][K|V][heads][slots][dim]
    side = H * P * D
    f8 = dtype == 4
    return L.PageView(K, V, KS if f8 else None, VS if f8 else None, pages * 2 * side, 2 * side, P * D, D,
                      layers * pages * 2 * side - side, layers, pages, H, P, D, dtype)


def sequences(L, rows=12, seqs=3, table_pages=5):
    return L.Sequences(TABLES, table_pages, LENS, STARTS, seqs, table_pages, rows, 0)


def attend_op(L, dtype=1, q_dtype=1, rows=12, G=2):
    v = view(L, dtype)
    hq = v.heads * G
    return L.PagedAttendOp(v, sequences(L, rows), Q, OUT, hq * 64, 64, hq * 64, 64, LSE, WORK, 1 << 30, 0.125, q_dtype, hq,
                           0, 0, 0, 0, 0)


def child_attend(lib, L, ctx, launches):
    call = lambda op: lib.pkv_paged_attend(ctx, C.byref(op), None)  # noqa: E731
    assert lib.pkv_paged_attend(None, C.byref(attend_op(L)), None) == INVALID and lib.pkv_paged_attend(ctx, None, None) == INVALID
    for dtype, qd in ((1, 1), (2, 2), (4, 1), (4, 2)):
        n = launches()
        assert call(attend_op(L, dtype, qd)) == OK and launches() > n
    before = launches()
    each(call, lambda: attend_op(L), [
        ("pages.dim", 96, UNSUPPORTED), ("pages.dim", 0, UNSUPPORTED), ("pages.dtype", 0, INVALID),
        ("pages.dtype", 3, INVALID), ("pages.dtype", 5, INVALID), ("pages.layers", 0, INVALID),
        ("pages.layers", 2, INVALID), ("pages.pages", 0, INVALID), ("pages.pages", 11, INVALID),
        ("pages.heads", 0, INVALID), ("pages.heads", 3, INVALID), ("pages.page_slots", 8, INVALID),
        ("pages.page_slots", 33, INVALID), ("pages.page_slots", 64, INVALID), ("pages.page_slots", 1 << 17, INVALID),
        ("pages.d_keys", None, INVALID), ("pages.d_values", V + 8, INVALID), ("pages.d_key_scales", KS, INVALID),
        ("pages.slot_stride", 65, INVALID), ("pages.slot_stride", (1 << 22) + 8, INVALID), ("pages.elems", 100, INVALID),
        ("pages.page_stride", 1 << 62, INVALID), ("pages.head_stride", 12, INVALID),
        ("seqs.d_tables", None, INVALID), ("seqs.d_tables", TABLES + 2, INVALID), ("seqs.d_lens", None, INVALID),
        ("seqs.d_lens", LENS + 1, INVALID), ("seqs.d_starts", STARTS + 2, INVALID), ("seqs.seqs", 0, INVALID),
        ("seqs.seqs", (1 << 24) + 1, INVALID), ("seqs.table_pages", 0, INVALID), ("seqs.table_pages", 1 << 26, INVALID),
        ("seqs.table_stride", 1 << 62, INVALID), ("seqs.reserved", 1, INVALID), ("seqs.rows", 1 << 29, INVALID),
        ("d_q", None, INVALID), ("d_q", Q + 4, INVALID), ("d_out", None, INVALID), ("d_out", OUT + 8, INVALID),
        ("d_out", Q, INVALID), ("d_out", Q + 1024, INVALID), ("d_out", K + 4096, INVALID), ("d_out", V, INVALID), ("q_row_stride", 257, INVALID),
        ("q_head_stride", 1 << 62, INVALID), ("out_head_stride", 56, INVALID), ("out_row_stride", 64, INVALID),
        ("d_lse", LSE + 2, INVALID), ("d_workspace", None, INVALID), ("d_workspace", WORK + 64, INVALID),
        ("workspace_bytes", 0, CAPACITY), ("scale", 0.0, INVALID), ("scale", -1.0, INVALID),
        ("scale", float("nan"), INVALID), ("scale", float("inf"), INVALID), ("scale", 3e38, INVALID),
        ("dtype", 0, INVALID), ("dtype", 2, INVALID), ("dtype", 4, INVALID), ("q_heads", 0, INVALID),
        ("q_heads", 3, INVALID), ("max_len", 161, INVALID), ("clear", 2, INVALID)])
    each(call, lambda: attend_op(L, 4, 1), [
        ("pages.d_key_scales", None, INVALID), ("pages.d_value_scales", None, INVALID),
        ("pages.d_key_scales", KS + 8, INVALID), ("pages.slot_stride", 128, INVALID),
        ("pages.head_stride", 32 * 64 - 64, INVALID), ("dtype", 0, INVALID)])
    assert launches() == before
    op = attend_op(L, rows=0)
    assert call(op) == OK and launches() == before
    op = attend_op(L, rows=13)      # not as many for each of 3
    op.seqs.d_starts = None
    assert call(op) == INVALID and lib.pkv_paged_attend_workspace(C.byref(op)) == 0
    size = lib.pkv_paged_attend_workspace(C.byref(attend_op(L)))
    op = attend_op(L)
    op.workspace_bytes = size - 1
    assert size and call(op) == CAPACITY and launches() == before
    # the workspace's size needs no address
    bare = attend_op(L)
    bare.pages.d_keys = bare.pages.d_values = bare.seqs.d_tables = bare.seqs.d_lens = bare.d_q = bare.d_out = None
    assert lib.pkv_paged_attend_workspace(C.byref(bare)) == size and lib.pkv_paged_attend_workspace(None) == 0
    each(call, lambda: attend_op(L), [("seqs.d_starts", None, OK), ("d_lse", None, OK), ("max_len", 160, OK), ("max_len", 1, OK),
                                      ("max_rows", 2 ** 32 - 1, OK), ("window", 2 ** 32 - 1, OK), ("sinks", 2 ** 32 - 1, OK),
                                      ("clear", 1, OK), ("seqs.table_stride", 0, OK), ("pages.page_stride", 0, OK),
                                      ("q_head_stride", 0, OK)])


def rows_op(L, dtype=1, cache=4, rows=12, layers=3):
    v = view(L, cache, layers=layers)
    return L.PagedRowsOp(v, sequences(L, rows), Q, OUT, max(rows, 1) * 128, 128, 64, dtype, 0)


def child_rows(lib, L, ctx, launches):
    for store, entry in ((True, lib.pkv_paged_store), (False, lib.pkv_paged_load)):
        call = lambda op: entry(ctx, C.byref(op), None)  # noqa: E731,B023
        assert entry(None, C.byref(rows_op(L)), None) == INVALID and entry(ctx, None, None) == INVALID
        for cache in (1, 2, 4):
            for dtype in (0, 1, 2):
                n = launches()
                assert call(rows_op(L, dtype, cache)) == OK and launches() > n
        before = launches()
        each(call, lambda: rows_op(L), [
            ("pages.dtype", 0, INVALID), ("pages.dim", 32, UNSUPPORTED), ("pages.elems", 100, INVALID),
            ("pages.d_keys", None, INVALID), ("pages.d_value_scales", None, INVALID), ("pages.heads", (1 << 16) + 1, INVALID),
            ("dtype", 3, INVALID), ("dtype", 4, INVALID), ("dtype", -1, INVALID), ("reserved", 1, INVALID),
            ("seqs.d_tables", None, INVALID), ("seqs.d_lens", None, INVALID), ("seqs.rows", 1 << 31, INVALID),
            ("d_keys", Q + 2, INVALID), ("d_values", OUT + 4, INVALID), ("row_stride", 63, INVALID),
            ("layer_stride", 1 << 63, INVALID)])
        assert launches() == before
        # rows on the pages or their scales, and a load of both sides into one place
        each(call, lambda: rows_op(L), [("d_keys", K + 4096, INVALID), ("d_values", V, INVALID), ("d_keys", VS, INVALID),
                                        ("d_values", KS + 16, INVALID), ("d_values", Q + 1024, OK if store else INVALID)])
        # what is written has no two rows in one place
        each(call, lambda: rows_op(L), [("pages.layer_stride", 0, INVALID if store else OK),
                                        ("layer_stride", 0, OK if store else INVALID)])
        before = launches()
        assert call(rows_op(L, rows=0)) == OK
        op = rows_op(L)
        op.d_keys = op.d_values = None
        assert call(op) == OK and launches() == before
        op = rows_op(L, layers=1)
        op.layer_stride, op.seqs.rows, op.row_stride = 0, 3 << 26, 128        # 2^24 chunks of 16 rows and more
        op.d_keys, op.d_values = 1 << 50, 1 << 51
        assert call(op) == OK
        op.seqs.rows = (1 << 28) + 1
        assert call(op) == INVALID
        each(call, lambda: rows_op(L), [("d_keys", None, OK), ("d_values", None, OK), ("seqs.d_starts", None, OK)])


def prompts_op(L, dtype=1, rows=50, H=2, G=3, D=64):
    w = (H * G + 2 * H) * D
    return L.PromptsOp(Q, Q + 2 * H * G * D, Q + 2 * (H * G + H) * D, OUT, w, D, w, D, w, D, H * G * D, D, STARTS, LSE, WORK,
                       1 << 30, 0.125, dtype, 4, rows, H, H * G, D, 0, 0, 0, 0)


def child_prompts(lib, L, ctx, launches):
    call = lambda op: lib.pkv_prompts(ctx, C.byref(op), None)  # noqa: E731
    assert lib.pkv_prompts(None, C.byref(prompts_op(L)), None) == INVALID and lib.pkv_prompts(ctx, None, None) == INVALID
    for dtype in (1, 2):
        n = launches()
        assert call(prompts_op(L, dtype)) == OK and launches() > n
    before = launches()
    each(call, lambda: prompts_op(L), [
        ("dim", 96, UNSUPPORTED), ("dtype", 0, INVALID), ("dtype", 3, INVALID), ("dtype", 4, INVALID), ("heads", 0, INVALID),
        ("heads", 4, INVALID), ("q_heads", 0, INVALID), ("q_heads", 5, INVALID), ("seqs", 0, INVALID),
        ("seqs", (1 << 24) + 1, INVALID), ("rows", 1 << 30, INVALID), ("clear", 2, INVALID), ("d_starts", None, INVALID),
        ("d_starts", STARTS + 2, INVALID), ("d_q", None, INVALID), ("d_k", None, INVALID), ("d_v", None, INVALID),
        ("d_out", None, INVALID), ("d_k", Q + 2, INVALID), ("d_v", Q + 8, INVALID), ("d_out", Q, INVALID),
        ("k_row_stride", 100, INVALID), ("v_head_stride", 60, INVALID), ("k_row_stride", (1 << 22) + 8, INVALID),
        ("out_row_stride", 64, INVALID), ("out_head_stride", 0, INVALID), ("d_lse", LSE + 1, INVALID),
        ("scale", 0.0, INVALID), ("scale", float("inf"), INVALID)])
    assert call(prompts_op(L, rows=0)) == OK and launches() == before
    op = prompts_op(L)
    need = lib.pkv_prompts_workspace(C.byref(op))
    if need:
        op.workspace_bytes = need - 1
        assert call(op) == CAPACITY
    op.q_heads = 5
    assert lib.pkv_prompts_workspace(C.byref(op)) == 0 and lib.pkv_prompts_workspace(None) == 0
    each(call, lambda: prompts_op(L), [("d_lse", None, OK), ("max_rows", 2 ** 32 - 1, OK), ("window", 2 ** 32 - 1, OK),
                                       ("clear", 1, OK), ("q_head_stride", 0, OK), ("k_head_stride", 0, OK)])


def child_sizes(lib, L, ctx, launches):
    """Large calls are taken, and those past a launch's size refused, by sizes alone."""
    def call(rows, seqs, heads, G, each_row=False, table_pages=1 << 12, page=64):
        op = attend_op(L)
        v = op.pages
        v.heads, v.page_slots, v.head_stride, v.page_stride, v.pages, v.elems = heads, page, 0, 0, 1, page * 64
        op.seqs.rows, op.seqs.seqs, op.seqs.table_pages, op.seqs.table_stride = rows, seqs, table_pages, 0
        op.q_heads = heads * G
        op.q_row_stride = op.q_head_stride = 0
        op.d_q, op.d_out = 1 << 55, 1 << 56
        op.out_head_stride, op.out_row_stride = 64, heads * G * 64
        op.workspace_bytes = 1 << 62
        if each_row:
            op.seqs.d_starts = None
        need, n = lib.pkv_paged_attend_workspace(C.byref(op)), launches()
        rc = lib.pkv_paged_attend(ctx, C.byref(op), None)
        assert rc in (OK, INVALID) and (launches() > n) == (rc == OK), rc
        assert rc == OK or need == 0
        assert need < 1 << 36, need
        return rc == OK

    assert call(64, 64, 8, 8, True) and call(1 << 16, 1 << 16, 8, 4, True) and call(1 << 20, 64, 8, 4)
    assert call(1 << 25, 256, 8, 4) and not call((1 << 25) + 1, 256, 8, 4)          # rows x query heads
    assert call(1 << 17, 1 << 17, 16, 1, True) and not call(1 << 21, 1 << 21, 16, 1, True)
    assert call(3, 3, 1 << 16, 1, True) and not call(3, 3, (1 << 16) + 1, 1, True)
    assert call(64, 64, 8, 8, True, table_pages=1 << 13, page=65536) and not call(64, 64, 8, 8, True, table_pages=1 << 14,
                                                                                  page=65536)


def test_python_refusals():
    import torch
    from provekv_amd.paged import PagedKVCache, attend_prompts
    from provekv_amd.pool import PagedKVCache as Same
    assert Same is PagedKVCache
    cache = PagedKVCache(2, 2, 6, 16, 64, device="cpu")
    small = PagedKVCache(2, 2, 6, 16, 64, dtype=torch.float8_e4m3fn, device="cpu")
    assert cache.buf.dtype == torch.bfloat16 and small.buf.dtype == torch.uint8 and small.scales.shape[-1] == 2
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    starts = torch.tensor([0, 2, 3, 6], dtype=torch.int32)
    q = torch.zeros(6, 4, 64, dtype=torch.bfloat16)
    good = (0, q, tables, lens)
    for err, args, kw in (
            (TypeError, (0, q.float(), tables, lens), {}), (TypeError, (0, q.half(), tables, lens), {}),
            (ValueError, (0, q[0], tables, lens), {}), (ValueError, (0, q[..., :32], tables, lens), {}),
            (ValueError, (0, q[:, :3], tables, lens), {}), (ValueError, (0, q[:, :0], tables, lens), {}),
            (ValueError, (0, q[:5], tables, lens), {}), (ValueError, (0, q, tables[0], lens), {}),
            (ValueError, (0, q, tables.long(), lens), {}), (ValueError, (0, q, tables[:0], lens), {}),
            (ValueError, (0, q, tables.t().contiguous().t(), lens), {}), (IndexError, (2, q, tables, lens), {}),
            (ValueError, (0, q.clone().requires_grad_(), tables, lens), {}), (ValueError, good, dict(window=-1)),
            (ValueError, good, dict(sinks=-1)), (ValueError, good, dict(max_rows=0)), (ValueError, good, dict(max_len=0)),
            (ValueError, good, dict(max_len=33)), (ValueError, good, dict(out=q.float())),
            (ValueError, good, dict(lse=torch.zeros(6, 4))), (ValueError, good, dict(starts=starts)),
            (ValueError, good, {})):                                           # the last two: not on a GPU
        with pytest.raises(err):
            cache.attend(*args, **kw)
    with pytest.raises(TypeError):
        small.attend(0, q.float(), tables, lens)
    rows = torch.zeros(2, 6, 2, 64)
    for err, args in ((TypeError, (rows, rows.half())), (TypeError, (rows.double(), None)), (ValueError, (rows, rows[:, :5])),
                      (ValueError, (rows[:1], None)), (ValueError, (rows[..., :32], None)), (ValueError, (rows[0], None)),
                      (ValueError, (rows.clone().requires_grad_(), None)), (ValueError, (rows, rows))):
        with pytest.raises(err):
            small.store(*args, tables, lens)
    assert small.store(None, None, tables, lens) is None
    with pytest.raises(TypeError):
        small.load(6, tables, lens, dtype=torch.float64)
    with pytest.raises(ValueError):
        small.load(-1, tables, lens)
    buf = torch.zeros(2, 6, 2, 2, 16, 64, dtype=torch.uint8)
    for err, args in ((TypeError, (buf.int(),)), (ValueError, (buf,)), (ValueError, (buf.to(torch.float16), small.scales)),
                      (ValueError, (buf[:, :, :1], small.scales)), (ValueError, (buf, small.scales[..., :1])),
                      (ValueError, (buf, small.scales.float())), (ValueError, (buf[..., :32].contiguous(), small.scales)),
                      (ValueError, (buf[..., :8, :].contiguous(), small.scales)), (ValueError, (buf.transpose(0, 1), small.scales))):
        with pytest.raises(err):
            PagedKVCache.over(*args)
    k = q[:, :2]
    for err, args, kw in (
            (TypeError, (q.float(), k.float(), k.float(), starts), {}), (TypeError, (q, k.half(), k, starts), {}),
            (ValueError, (q, k[:5], k[:5], starts), {}), (ValueError, (q, q[:, :3], q[:, :3], starts), {}),
            (ValueError, (q, k, q[:, :1], starts), {}), (ValueError, (q[..., :32], k[..., :32], k[..., :32], starts), {}),
            (ValueError, (q, k, k, starts[:1]), {}), (ValueError, (q, k, k, starts), dict(window=-1)),
            (ValueError, (q, k.clone().requires_grad_(), k, starts), {}), (ValueError, (q, k, k, starts), {})):
        with pytest.raises(err):
            attend_prompts(*args, **kw)


if __name__ == "__main__":
    hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)   # found ahead of the runtime's own
    hip.host_hip_launched.restype = C.c_char_p
    from provekv_amd import _lib
    lib = _lib.lib()
    ctx = C.c_void_p()
    assert lib.pkv_ctx_create(0, C.byref(ctx)) == 0
    globals()["child_" + sys.argv[2]](lib, _lib, ctx, lambda: len(hip.host_hip_launched().split()))

"""The live-cache calls' argument checks, on the CPU: the C entries with the HIP
runtime replaced by tests/host_live_hip.cpp (no pointer is followed there), and
the Python methods on caches in host memory."""
import ctypes as C
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
OK, INVALID, CAPACITY, UNSUPPORTED = 0, 1, 11, 6


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("host_live") / "libhost_hip.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include",
                    os.path.join(HERE, "host_live_hip.cpp"), "-o", so], check=True)
    return so


@pytest.mark.parametrize("name", ["attend", "rows", "evict"])
def test_refusals(stub, name):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, name], capture_output=True, text=True,
                       timeout=120, env={**os.environ, "PYTHONPATH": os.path.dirname(HERE)})
    assert r.returncode == 0, r.stdout + r.stderr


K, V, KS, VS, Q, OUT, WORDS, WORDS2, W, W2, WORK, KEPT, LSE = (0x10000000 * (i + 1) for i in range(13))


def view(L, dtype=1, C_=2, layers=1, H=2, T=100, D=64):
    # keys and values of [copies][layers][K|V][heads][slots][dim]
    side = H * T * D
    fp4 = dtype == 3
    return L.KvView(K, V, KS if fp4 else None, VS if fp4 else None, layers * 2 * side, 2 * side, T * D, D,
                    C_ * layers * 2 * side - side, C_, layers, H, T, D, dtype)


def attend_op(L, dtype=1, q_dtype=1, n=3, G=2, **kw):
    v = view(L, dtype)
    hq = v.heads * G
    return L.AttendOp(v, Q, OUT, n * hq * 64, hq * 64, 64, n * hq * 64, hq * 64, 64, WORDS, WORDS2, LSE, W, 200, 100, WORK,
                      1 << 30, 0.125, q_dtype, hq, n, 0, 0, 0, 0)


def put(op, path, value):
    *front, last = path.split(".")
    for p in front:
        op = getattr(op, p)
    setattr(op, last, value)


def each(call, make, cases):
    for path, value, want in cases:
        op = make()
        put(op, path, value)
        got = call(op)
        assert got == want, (path, value, got)


def child_attend(lib, L, ctx, launches):
    call = lambda op: lib.pkv_attend(ctx, C.byref(op), None)  # noqa: E731
    assert lib.pkv_attend(None, C.byref(attend_op(L)), None) == INVALID and lib.pkv_attend(ctx, None, None) == INVALID
    for dtype, qd in ((0, 0), (1, 1), (2, 2), (3, 0), (3, 1), (3, 2)):
        n = launches()
        assert call(attend_op(L, dtype, qd)) == OK and launches() > n
    before = launches()
    common = [
        ("cache.dim", 96, UNSUPPORTED), ("cache.dim", 0, UNSUPPORTED), ("cache.dtype", 4, INVALID),
        ("cache.dtype", -1, INVALID), ("cache.copies", 0, INVALID), ("cache.layers", 0, INVALID),
        ("cache.layers", 2, INVALID), ("cache.heads", 0, INVALID), ("cache.slots", 0, INVALID),
        ("cache.slots", 101, INVALID), ("cache.slots", 0x7fffffff, INVALID), ("cache.d_keys", None, INVALID),
        ("cache.d_values", None, INVALID), ("cache.d_keys", K + 8, INVALID), ("cache.d_values", V + 2, INVALID),
        ("cache.copy_stride", 2 ** 63, INVALID), ("cache.slot_stride", 65, INVALID), ("cache.elems", 38399, INVALID),
        ("d_q", None, INVALID), ("d_out", None, INVALID), ("d_q", Q + 4, INVALID), ("d_out", OUT + 8, INVALID),
        ("d_out", Q, INVALID), ("d_out", Q + 1024, INVALID), ("q_row_stride", 257, INVALID),
        ("q_copy_stride", 1 << 62, INVALID), ("out_head_stride", 63, INVALID), ("out_head_stride", 56, INVALID),
        ("out_row_stride", 64, INVALID), ("out_copy_stride", 0, INVALID), ("d_lens", None, INVALID),
        ("d_lens", WORDS + 2, INVALID), ("d_q_lens", WORDS + 1, INVALID), ("d_lse", LSE + 2, INVALID),
        ("d_weights", W + 1, INVALID), ("weight_head_stride", 99, INVALID), ("weight_copy_stride", 100, INVALID),
        ("d_workspace", None, INVALID), ("d_workspace", WORK + 64, INVALID), ("workspace_bytes", 0, CAPACITY),
        ("scale", 0.0, INVALID), ("scale", -1.0, INVALID), ("scale", float("nan"), INVALID),
        ("scale", float("inf"), INVALID), ("dtype", 2, INVALID), ("dtype", 3, INVALID), ("dtype", -1, INVALID),
        ("q_heads", 0, INVALID), ("q_heads", 3, INVALID), ("q_heads", 1, INVALID), ("nq", 0x7fffffff, INVALID), ("nq", 1 << 30, INVALID), ("scale", 3e38, INVALID),
        ("max_len", 101, INVALID), ("reserved", 1, INVALID), ("cache.d_key_scales", KS, INVALID)]
    each(call, lambda: attend_op(L), common)
    before = launches()
    each(call, lambda: attend_op(L, 3, 1), [
        ("cache.d_key_scales", None, INVALID), ("cache.d_value_scales", None, INVALID),
        ("cache.d_key_scales", KS + 1, INVALID), ("cache.d_value_scales", VS + 2, OK), ("cache.slot_stride", 32, INVALID), ("dtype", 3, INVALID)])
    before = launches()
    op = attend_op(L)
    op.nq = 0
    assert call(op) == OK and launches() == before
    size = lib.pkv_attend_workspace(C.byref(attend_op(L)))
    op = attend_op(L)
    op.workspace_bytes = size - 1
    assert size and call(op) == CAPACITY
    op.q_heads = 3
    assert lib.pkv_attend_workspace(C.byref(op)) == 0 and lib.pkv_attend_workspace(None) == 0
    # more workgroups than a launch holds
    op = attend_op(L, n=1, G=1)
    op.cache.heads = op.q_heads = 1 << 24
    op.cache.head_stride, op.q_head_stride, op.out_head_stride, op.d_weights = 0, 0, 64, None
    op.out_copy_stride = 1 << 30
    assert call(op) == INVALID and lib.pkv_attend_workspace(C.byref(op)) == 0
    each(call, lambda: attend_op(L), [("d_q_lens", None, OK), ("d_lse", None, OK), ("d_weights", None, OK),
                                      ("max_len", 100, OK), ("window", 2 ** 32 - 1, OK), ("sinks", 2 ** 32 - 1, OK),
                                      ("cache.copy_stride", 0, OK), ("q_head_stride", 0, OK)])


def rows_op(L, dtype=1, n=5):
    v = view(L, 3, layers=3)
    return L.RowsOp(v, Q, OUT, 3 * 2 * n * 64, 2 * n * 64, n * 64, 64, WORDS, WORDS2, dtype, n)


def child_rows(lib, L, ctx, launches):
    for store, entry in ((True, lib.pkv_fp4_store), (False, lib.pkv_fp4_load)):
        call = lambda op: entry(ctx, C.byref(op), None)  # noqa: E731,B023
        assert entry(None, C.byref(rows_op(L)), None) == INVALID and entry(ctx, None, None) == INVALID
        for dtype in (0, 1, 2):
            n = launches()
            assert call(rows_op(L, dtype)) == OK and launches() > n
        before = launches()
        each(call, lambda: rows_op(L), [
            ("cache.dtype", 1, INVALID), ("cache.dim", 32, UNSUPPORTED), ("cache.elems", 100, INVALID),
            ("cache.d_keys", None, INVALID), ("cache.d_value_scales", None, INVALID), ("dtype", 3, INVALID),
            ("dtype", -1, INVALID), ("d_first", None, INVALID), ("d_first", WORDS + 2, INVALID),
            ("d_counts", WORDS + 3, INVALID), ("d_keys", Q + 2, INVALID), ("d_values", OUT + 4, INVALID),
            ("row_stride", 63, INVALID), ("copy_stride", 1 << 63, INVALID), ("rows", 0x7fffffff, INVALID)])
        # what is written has no two rows in one place
        each(call, lambda: rows_op(L), [("cache.copy_stride", 0, INVALID if store else OK),
                                        ("copy_stride", 0, OK if store else INVALID)])
        before = launches()
        each(call, lambda: rows_op(L), [("rows", 0, OK)])
        op = rows_op(L)
        op.d_keys = op.d_values = None
        assert call(op) == OK and launches() == before
        op = rows_op(L)
        op.rows = 1 << 29
        op.copy_stride, op.layer_stride, op.head_stride = 1 << 40, 1 << 38, 1 << 36
        assert call(op) == INVALID and launches() == before
        each(call, lambda: rows_op(L), [("d_keys", None, OK), ("d_values", None, OK), ("d_counts", None, OK)])


def evict_op(L, dtype=1, in_place=False):
    v, t = view(L, dtype, layers=3), view(L, dtype, layers=3, T=40)
    t.d_keys, t.d_values = Q, OUT
    if dtype == 3:
        t.d_key_scales, t.d_value_scales = LSE, WORK
    if in_place:
        t = view(L, dtype, layers=3)
    return L.EvictOp(v, t, WORDS, WORDS2, KEPT, W, W if in_place else W2, (C.c_uint64 * 3)(600, 200, 100),
                     (C.c_uint64 * 3)(*((600, 200, 100) if in_place else (240, 80, 40))), 40, 4, 10, 0)


def child_evict(lib, L, ctx, launches):
    call = lambda op: lib.pkv_evict(ctx, C.byref(op), None)  # noqa: E731
    assert lib.pkv_evict(None, C.byref(evict_op(L)), None) == INVALID and lib.pkv_evict(ctx, None, None) == INVALID
    for dtype in (0, 1, 2, 3):
        for in_place in (False, True):
            n = launches()
            assert call(evict_op(L, dtype, in_place)) == OK and launches() > n
    before = launches()
    each(call, lambda: evict_op(L), [
        ("cache.dim", 1, UNSUPPORTED), ("into.dim", 128, INVALID), ("into.dtype", 2, INVALID), ("into.copies", 1, INVALID),
        ("into.layers", 2, INVALID), ("into.heads", 1, INVALID), ("into.slots", 39, INVALID), ("budget", 0, INVALID),
        ("budget", 41, INVALID), ("budget", 13, INVALID), ("sinks", 31, INVALID), ("recent", 37, INVALID),
        ("recent", 2 ** 32 - 1, INVALID), ("sinks", 2 ** 32 - 1, INVALID), ("d_lens", None, INVALID),
        ("d_new_lens", None, INVALID), ("d_new_lens", WORDS, INVALID), ("d_new_lens", WORDS + 4, INVALID),
        ("d_kept", None, INVALID), ("d_weights", None, INVALID), ("d_weights_out", None, INVALID),
        ("d_weights_out", W, INVALID), ("d_weights_out", W + 400, INVALID), ("d_kept", KEPT + 2, INVALID),
        ("into.d_keys", K, INVALID), ("into.d_keys", K + 128, INVALID), ("into.d_values", K + 128, INVALID),
        ("into.slot_stride", 0, INVALID), ("reserved", 1, INVALID)])
    op = evict_op(L)
    op.out_strides[2] = 39
    assert call(op) == INVALID
    op = evict_op(L, in_place=True)
    op.out_strides[0] = 1200          # one memory, other places
    assert call(op) == INVALID and launches() == before
    op = evict_op(L, in_place=True)
    op.cache.copy_stride = op.into.copy_stride = 0
    assert call(op) == INVALID
    op = evict_op(L)
    op.cache.heads = op.into.heads = 1 << 20
    op.cache.elems = op.into.elems = 1 << 60
    op.cache.head_stride, op.cache.layer_stride, op.cache.copy_stride = 0, 0, 0
    op.into.head_stride, op.into.layer_stride, op.into.copy_stride = 1 << 16, 1 << 40, 1 << 44
    op.into.d_keys, op.into.d_values = 1 << 50, 1 << 58
    op.out_strides[2], op.out_strides[1], op.out_strides[0] = 40, 1 << 30, 1 << 34
    op.weight_strides[0] = op.weight_strides[1] = op.weight_strides[2] = 0
    op.d_weights_out = 1 << 59
    assert call(op) == INVALID


def test_python_refusals():
    import torch
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    cache = DeviceKVCache(2, 2, 10, 64, dtype=torch.bfloat16, copies=2, device="cpu")
    four = FourBitKVCache(2, 2, 10, 64, copies=2, device="cpu")
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    lens = torch.zeros(2, dtype=torch.int32)
    for err, args, kw in (
            (TypeError, (0, q.float(), lens), {}), (TypeError, (0, q.double(), lens), {}),
            (ValueError, (0, q[0], lens), {}), (ValueError, (0, q[:1], lens), {}), (ValueError, (0, q[..., :32], lens), {}),
            (ValueError, (0, q[:, :, :3], lens), {}), (ValueError, (0, q[:, :, :0], lens), {}),
            (ValueError, (0, q.clone().requires_grad_(), lens), {}), (ValueError, (0, q, lens), dict(window=-1)),
            (ValueError, (0, q, lens), dict(sinks=-1)), (ValueError, (0, q, lens), {})):   # the last: not on a GPU
        with pytest.raises(err):
            cache.attend(*args, **kw)
    with pytest.raises(TypeError):
        four.attend(0, q.double(), lens)
    w = torch.zeros(2, 2, 2, 10)
    other = DeviceKVCache(2, 2, 4, 64, dtype=torch.bfloat16, copies=2, device="cpu")
    for kw in (dict(budget=0), dict(budget=5, sinks=3, recent=3), dict(budget=5, sinks=-1), dict(budget=5, into=other),
               dict(budget=4, into=four), dict(budget=5, layer=0), dict(budget=5)):
        with pytest.raises(ValueError):
            cache.evict(lens, w, **kw)
    with pytest.raises(ValueError):
        cache.evict(lens, w.double(), 5)
    rows = torch.zeros(2, 2, 2, 3, 64)
    for err, args in ((TypeError, (rows, rows.half(), 0)), (TypeError, (rows.double(), None, 0)),
                      (ValueError, (rows, rows[:, :, :, :2], 0)), (ValueError, (rows[:, :1], None, 0)),
                      (ValueError, (rows, rows, 0))):
        with pytest.raises(err):
            four.store(*args)
    assert four.store(None, None, 0) is None
    with pytest.raises(TypeError):
        four.load(0, 1, dtype=torch.float64)
    with pytest.raises(ValueError):
        FourBitKVCache(1, 1, 4, 96, device="cpu")
    for bad in (torch.zeros(2, 2, 1, 2, 10, 64), torch.zeros(2, 2, 2, 10, 64), torch.zeros(2, 2, 2, 2, 10, 128)[..., :64]):
        with pytest.raises(ValueError):
            DeviceKVCache.over(bad)
    with pytest.raises(ValueError):
        FourBitKVCache.over(four.codes, four.scales[..., :1])


if __name__ == "__main__":
    hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)   # found ahead of the runtime's own
    hip.host_hip_launched.restype = C.c_char_p
    from provekv_amd import _lib
    lib = _lib.lib()
    ctx = C.c_void_p()
    assert lib.pkv_ctx_create(0, C.byref(ctx)) == 0
    globals()["child_" + sys.argv[2]](lib, _lib, ctx, lambda: len(hip.host_hip_launched().split()))

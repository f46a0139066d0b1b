"""Sizes at which the live-cache calls begin to refuse, on the CPU: both sides of
every limit that include/pkv_codec.h names, by the C entries with the HIP
runtime replaced by tests/host_live_hip.cpp (no pointer is followed there)."""
import ctypes as C
import os
import subprocess
import sys

import pytest

from test_live_host import INVALID, OK, attend_op, evict_op, stub  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.parametrize("name", ["attend", "evict"])
def test_limits(stub, name):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub, name], capture_output=True, text=True,
                       timeout=120, env={**os.environ, "PYTHONPATH": os.pathsep.join((os.path.dirname(HERE), HERE))})
    assert r.returncode == 0, r.stdout + r.stderr


def attend(L, copies, heads, q_heads, nq, slots, weights, dim=128, dtype=1, window=0):
    """A call over one memory for all copies and heads (what is only read may
    share it); outputs and weights apart."""
    op = attend_op(L, dtype, dtype)
    v = op.cache
    v.copies, v.heads, v.slots, v.dim = copies, heads, slots, dim
    v.copy_stride = v.layer_stride = v.head_stride = 0
    v.slot_stride, v.elems = dim, slots * dim
    op.q_heads, op.nq, op.window, op.max_len = q_heads, nq, window, 0
    op.d_q, op.d_out = 1 << 55, 1 << 56
    op.q_copy_stride = op.q_row_stride = op.q_head_stride = 0
    op.out_head_stride, op.out_row_stride, op.out_copy_stride = dim, q_heads * dim, nq * q_heads * dim
    op.d_weights = (1 << 54) if weights else None
    op.weight_head_stride, op.weight_copy_stride = slots, heads * slots
    op.workspace_bytes = (1 << 62)
    return op


def child_attend(lib, L, ctx, launches):
    def call(*args, **kw):
        op = attend(L, *args, **kw)
        need, n = lib.pkv_attend_workspace(C.byref(op)), launches()
        rc = lib.pkv_attend(ctx, C.byref(op), None)
        assert rc in (OK, INVALID) and (launches() > n) == (rc == OK), rc
        # sizes alone decide, so the workspace's answer goes with the call's
        assert rc == OK or need == 0, (args, need)
        return rc == OK

    # long prompts of many agents and heads: millions of rows in thousands of workgroups
    assert call(1, 128, 128, 131072, 131072, True) and call(64, 32, 32, 8192, 8192, True)
    assert call(8, 8, 64, 32768, 32768, False) and call(16, 32, 32, 32768, 32768, False)
    assert call(16, 32, 32, 32768, 32768, True, dtype=0, dim=64)
    # copies x query heads x rows
    assert call(1, 64, 64, 1 << 24, 1 << 24, False) and not call(1, 64, 64, (1 << 24) + 1, 1 << 25, False)
    # up to 16 rows of a head: a workgroup a row joins its shares
    most = (1 << 24) - 1
    assert call(1, most, most, 1, 64, False) and not call(1, most + 1, most + 1, 1, 64, False)
    quarter = most // 4
    assert call(1, quarter, quarter * 4, 1, 64, False) and not call(1, quarter + 1, quarter * 4 + 4, 1, 64, False)
    # .. and 1,024 slots a workgroup with weights
    assert call(1, most // 2, most // 2, 1, 1024, True) and not call(1, most // 2 + 1, most // 2 + 1, 1, 1024, True)
    assert call(1, most // 5, most // 5, 1, 4000, True) and not call(1, most // 5 + 1, most // 5 + 1, 1, 4000, True)
    # more rows: their tiles
    assert call(1, most, most, 17, 64, False) and not call(1, most + 1, most + 1, 17, 64, False)
    # .. and with weights blocks of 128 slots, no more than a window's
    assert call(1, most // 8, most // 8, 17, 1024, True) and not call(1, most // 7, most // 7, 17, 1024, True)
    assert call(1, most // 8, most // 8, 17, 100000, True, window=100)


def evict(L, dtype, dim, heads, budget, in_place):
    """One copy and layer of `heads` heads, rows a head apart."""
    op = evict_op(L, dtype, in_place)
    slots = budget + 10
    for v in (op.cache, op.into):
        v.copies = v.layers = 1
        v.heads, v.slots, v.dim, v.slot_stride, v.head_stride = heads, slots, dim, dim, slots * dim
        v.elems = heads * slots * dim
    op.cache.d_keys, op.cache.d_values = 1 << 50, 1 << 51
    op.into.d_keys, op.into.d_values = (1 << 50, 1 << 51) if in_place else (1 << 52, 1 << 53)
    if dtype == 3:
        op.cache.d_key_scales, op.cache.d_value_scales = 1 << 54, 1 << 55
        op.into.d_key_scales, op.into.d_value_scales = (1 << 54, 1 << 55) if in_place else (1 << 56, 1 << 57)
    op.d_weights = 1 << 58
    op.d_weights_out = 1 << (58 if in_place else 59)
    op.weight_strides[2] = op.out_strides[2] = slots
    op.budget, op.sinks, op.recent = budget, 0, 0
    return op


def child_evict(lib, L, ctx, launches):
    def call(*args):
        op = evict(L, *args)
        n = launches()
        rc = lib.pkv_evict(ctx, C.byref(op), None)
        assert rc in (OK, INVALID) and (launches() > n) == (rc == OK), rc
        return rc == OK

    most = (1 << 24) - 1
    for dtype, size in ((0, 4), (1, 2), (2, 2), (3, 0.5)):
        for dim in (64, 128):
            row = int(dim * size)
            # in place: columns of 64 bytes of both sides, whatever the budget
            sets = min((1 << 22) - 1, most // (2 * max(row // 64, 1)))
            for budget in (1, 4096):
                assert call(dtype, dim, sets, budget, True) and not call(dtype, dim, sets + 1, budget, True)
            # into other memory: 16 KiB of rows
            rows = (1 << 14) // row
            assert call(dtype, dim, (1 << 22) - 1, rows, False) and not call(dtype, dim, 1 << 22, rows, False)
            for blocks in (7, 100):
                sets = most // (2 * blocks)
                assert call(dtype, dim, sets, rows * blocks, False)
                assert not call(dtype, dim, sets + 1, rows * blocks, False)
                assert not call(dtype, dim, sets, rows * blocks + 1, False)


if __name__ == "__main__":
    hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)   # found ahead of the runtime's own
    hip.host_hip_launched.restype = C.c_char_p
    from provekv_amd import _lib
    lib = _lib.lib()
    ctx = C.c_void_p()
    assert lib.pkv_ctx_create(0, C.byref(ctx)) == 0
    globals()["child_" + sys.argv[2]](lib, _lib, ctx, lambda: len(hip.host_hip_launched().split()))

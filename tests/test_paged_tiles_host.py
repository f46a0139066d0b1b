"""Which tile of the many-row attention kernel a call takes, on the CPU: the
kernels that the C entries launch with the HIP runtime replaced by
tests/host_live_hip.cpp; and the plain form that the GPU tests of those tiles go
by against the row-by-row one."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

import paged_ref as P
import paged_tiles as T
from test_live_host import stub  # noqa: F401

HERE = os.path.dirname(os.path.abspath(__file__))
TYPES = {1: (1,), 2: (2,), 4: (1, 2)}            # pages: queries


def test_launches(stub):  # noqa: F811
    r = subprocess.run([sys.executable, os.path.abspath(__file__), stub], capture_output=True, text=True, timeout=120,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join((os.path.dirname(HERE), HERE))})
    assert r.returncode == 0, r.stdout + r.stderr


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 2), (3, 40)])
def test_plain_form(window, sinks):
    g = torch.Generator().manual_seed(1)
    lens, spans = [50, 3, 0, 20], [(1, 30), (31, 5), (36, 2), (38, 1)]
    kv = []
    for n in lens:
        K, V = (torch.randn(2, n, 64, generator=g, dtype=torch.float64) for _ in range(2))
        kv.append((K, V, torch.rand(n, generator=g) < 0.8))
    kv[0][1][1, 30, 5], kv[0][1][0, 41, 6], kv[0][0][1, 45, 7] = math.inf, math.nan, math.nan
    q = torch.randn(40, 6, 64, generator=g, dtype=torch.float64)
    a, b = (f(q, kv, lens, spans, window, sinks, 0.125) for f in (T.attend, P.attend))
    for name in b:
        # the same sums of up to 50 terms in another order; NaN and infinities in the same places
        x, y = a[name], b[name]
        near = (x - y).abs() <= 1e-12 * (1 + y.abs())
        assert (near | (x == y) | (torch.isnan(x) & torch.isnan(y))).all(), name
    assert torch.isnan(b["out"]).any() and torch.isinf(b["out"]).any()


def kernels(hip, call):
    n = len(hip.host_hip_launched())
    assert call() == 0
    return hip.host_hip_launched()[n:].decode().split()


def expect(names, pages, queries, D, paged, rows, joined, what):
    want = f"rows_kernelILi{pages}ELi{queries}ELi{D}ELb{int(paged)}ELi{256 // rows}EE"
    assert sum("11rows_kernelI" in x for x in names) == 1 and any(want in x for x in names), (what, want, names)
    assert any("16join_rows_kernelI" in x for x in names) == joined, (what, names)


def counted(names):
    """Plan kernels ahead of the others."""
    return sum("plan_kernel" in x for x in names)


if __name__ == "__main__":
    hip = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)   # found ahead of the runtime's own
    hip.host_hip_launched.restype = C.c_char_p
    from provekv_amd import _lib as L
    lib, ctx = L.lib(), C.c_void_p()
    assert lib.pkv_ctx_create(0, C.byref(ctx)) == 0
    K, V, KS, VS, Q, OUT, TABLES, LENS, STARTS, WORK = (i << 44 for i in range(1, 11))
    for D in (64, 128):
        for name, (tile, joined, H, G, counts, lens, page, window, sinks) in T.PAGED.items():
            for pages, queries in ((p, q) for p, both in TYPES.items() for q in both):
                n, side, hq, rows = T.table_pages(lens, page), H * page * D, H * G, 5 + sum(counts)
                f8 = pages == 4
                v = L.PageView(K, V, KS if f8 else None, VS if f8 else None, 200 * 2 * side, 2 * side, page * D, D,
                               200 * 2 * side - side, 1, 200, H, page, D, pages)
                s = L.Sequences(TABLES, n, LENS, STARTS, len(counts), n, rows, 0)
                op = L.PagedAttendOp(v, s, Q, OUT, hq * D, D, hq * D, D, None, WORK, 1 << 40, 0.125, queries, hq, max(counts), 0,
                                     window, sinks, 0)
                got = kernels(hip, lambda: lib.pkv_paged_attend(ctx, C.byref(op), None))
                expect(got, pages, queries, D, True, tile, joined, name)
        for name, (tile, joined, H, G, counts, window, sinks) in T.PROMPTS.items():
            for dtype in (1, 2):
                hq, w = H * G, H * (G + 2) * D
                op = L.PromptsOp(Q, K, V, OUT, w, D, w, D, w, D, hq * D, D, STARTS, None, WORK, 1 << 40, 0.125, dtype, len(counts),
                                 5 + sum(counts), H, hq, D, max(counts), window, sinks, 0)
                got = kernels(hip, lambda: lib.pkv_prompts(ctx, C.byref(op), None))
                expect(got, dtype, dtype, D, False, tile, joined, name)
    # up to 256 sequences are counted by every workgroup, more by a kernel ahead of each that cuts them
    for seqs, ahead in ((1, 0), (64, 0), (256, 0), (257, 1), (5000, 1)):
        side = 2 * 16 * 64
        for starts, rows, most, kinds in ((None, seqs, 0, 1), (STARTS, seqs, 1, 1), (STARTS, seqs + 40, 0, 2)):
            v = L.PageView(K, V, None, None, 200 * 2 * side, 2 * side, 16 * 64, 64, 200 * 2 * side - side, 1, 200, 2, 16, 64, 1)
            s = L.Sequences(TABLES, 9, LENS, starts, seqs, 9, rows, 0)
            op = L.PagedAttendOp(v, s, Q, OUT, 128, 64, 128, 64, None, WORK, 1 << 40, 0.125, 1, 2, most, 0, 0, 0, 0)
            got = counted(kernels(hip, lambda: lib.pkv_paged_attend(ctx, C.byref(op), None)))
            assert got == kinds * ahead, (seqs, kinds, got)
        op = L.PromptsOp(Q, K, V, OUT, 384, 64, 384, 64, 384, 64, 128, 64, STARTS, None, WORK, 1 << 40, 0.125, 1, seqs, seqs + 40, 2,
                         2, 64, 0, 0, 0, 0)
        assert counted(kernels(hip, lambda: lib.pkv_prompts(ctx, C.byref(op), None))) == ahead

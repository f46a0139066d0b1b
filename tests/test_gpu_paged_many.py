"""Packed calls of more sequences than a wave counts for itself (256): units of
work from the plan kernels, rows found by a search; against the plain 64-bit
form, captured, with starts that do not ascend, and in time that grows with the
sequences and not with their square."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
import paged_tiles as T
from test_gpu_paged import BF16, F8, KIND_IDS, KINDS, make, running, words
from test_gpu_paged_rows import check as check_rows

pytestmark = pytest.mark.gpu


def run(cache, dtype, tables, lens, counts, G, starts=True, window=0, sinks=0, **kw):
    """As test_gpu_paged.run, a sequence of the plain form at a time; 2 and 3 rows of nobody."""
    before, behind = (2, 3) if starts else (0, 0)
    st = [before + x for x in running(counts)]
    rows = st[-1] + behind
    q = torch.randn(rows, cache.heads * G, cache.dim, generator=torch.Generator().manual_seed(71)).to(dtype)
    lse = torch.full((q.shape[1], rows), 77.0, device="cuda")
    out = torch.full(q.shape, 55.0, dtype=dtype, device="cuda")
    cache.attend(0, q.cuda(), words(tables), words(lens), starts=words(st) if starts else None, window=window, sinks=sinks,
                 lse=lse, out=out, **kw)
    spans = P.rows_of(st, len(lens), rows)
    some = [i for i in range(len(lens)) if lens[i] > 300 or i % 5 == 0 or i > len(lens) - 4]     # looked at
    pages = P.values(cache.buf, cache.scales)[0]
    kv = [P.gathered(pages, tables[i], lens[i]) for i in some]
    ref = T.attend(q.double(), kv, [lens[i] for i in some], [spans[i] for i in some], window, sinks, 1 / math.sqrt(cache.dim))
    P.check(out, lse, ref, [spans[i] for i in some], dtype)
    nobody = [i for i in range(rows) if i < before or i >= st[-1]]
    assert (out[nobody] == 55).all() and (lse[:, nobody] == 77).all()
    assert torch.isfinite(out).all() and not (out[before:st[-1]] == 55).any()
    new = cache.attend(0, q.cuda(), words(tables), words(lens), starts=words(st) if starts else None, window=window, sinks=sinks,
                       **kw)
    assert R.same(new[before:st[-1]], out[before:st[-1]]) and not new[nobody].any()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("seqs", [257, 1100])
def test_tokens(ctx, seqs, cache_type, dtype):
    """Single tokens; some of sequences long enough to be cut and joined."""
    lens = [3000 if i in (5, seqs - 2) else 1 + i * 37 % 90 for i in range(seqs)]
    cache, tables = make(cache_type, 1, 64, 16, lens, seed=70)
    run(cache, dtype, tables, lens, [1] * seqs, 2, starts=False)
    run(cache, dtype, tables, lens, [i % 3 for i in range(seqs)], 1)
    run(cache, dtype, tables, lens, [min(lens[i], i % 2) for i in range(seqs)], 2, max_rows=1, window=40, sinks=2)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
def test_tokens_and_chunks(ctx, cache_type, dtype):
    lens = [2500 if i in (3, 290) else 1 + i * 53 % 120 for i in range(300)]
    cache, tables = make(cache_type, 1, 128, 32, lens, seed=72)
    run(cache, dtype, tables, lens, [300 if n > 2000 else (i % 4) * 13 % (n + 1) for i, n in enumerate(lens)], 2)
    run(cache, dtype, tables, lens, [1 if n < 2000 else 90 for n in lens], 1, max_rows=90)
    run(cache, dtype, tables, lens, [0 if i % 7 else min(n, 40) for i, n in enumerate(lens)], 3, window=100, sinks=5)


@pytest.mark.parametrize("H", [1, 8])
@pytest.mark.parametrize("dtype", [BF16, torch.float16], ids=["bf16", "f16"])
def test_prompts(ctx, dtype, H):
    from provekv_amd.paged import attend_prompts
    counts = [1300 if i == 200 else i * 7 % 41 for i in range(400)]
    st = [2 + x for x in running(counts)]
    x = torch.randn(st[-1] + 3, 3 * H, 64, generator=torch.Generator().manual_seed(73)).to(dtype)
    d = x.cuda()
    for kw in ({}, {"max_rows": 1300}, {"window": 30, "sinks": 2}):
        out = attend_prompts(d[:, :H], d[:, H:2 * H], d[:, 2 * H:], words(st), **kw)
        spans = P.rows_of(st, 400, x.shape[0])
        some = [i for i in range(400) if i % 9 == 0 or i in (200, 399)]
        kv = [(x[a:a + m, H:2 * H].double().transpose(0, 1), x[a:a + m, 2 * H:].double().transpose(0, 1),
               torch.ones(m, dtype=torch.bool)) for a, m in (spans[i] for i in some)]
        ref = T.attend(x[:, :H].double(), kv, [counts[i] for i in some], [spans[i] for i in some], kw.get("window", 0),
                       kw.get("sinks", 0), 0.125)
        P.check(out, None, ref, [spans[i] for i in some], dtype)
        assert torch.isfinite(out).all() and not out[:2].any() and not out[st[-1]:].any()


@pytest.mark.parametrize("seqs", [257, 5000])
def test_rows(ctx, seqs):
    lens = [1 + i * 7 % 40 for i in range(seqs)]
    cache, tables = make(F8, 1, 64, 16, lens, seed=74)
    counts = [min(n, i % 4) for i, n in enumerate(lens)]
    g = torch.Generator().manual_seed(75)
    check_rows(cache, torch.randn(2, 1, 3 + sum(counts) + 4, 1, 64, generator=g), tables, lens, counts, before=3, behind=4)


def test_captured(ctx):
    """Replays with other lengths and starts against the same call made eagerly."""
    from provekv_amd.paged import attend_prompts
    seqs, g = 300, torch.Generator().manual_seed(76)
    cache, tables = make(BF16, 2, 64, 16, [200] * seqs, seed=77)
    t, n, st = words(tables), words([200] * seqs), words(list(range(0, 4 * seqs + 1, 4)))
    q = torch.randn(4 * seqs, 4, 64, generator=g).to(BF16).cuda()
    outs = [torch.zeros_like(q) for _ in range(3)]

    def step(outs):
        cache.attend(0, q, t, n, starts=st, out=outs[0])
        attend_prompts(q, q[:, :2], q[:, 2:], st, out=outs[1])
        cache.attend(0, q[:seqs], t, n, out=outs[2][:seqs])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(outs)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(outs)
    for i in range(4):
        n.copy_(torch.randint(0, 201, (seqs,), generator=g).int())
        cuts = torch.randint(0, 4 * seqs + 1, (seqs + 1,), generator=g).sort()[0].int()
        st.copy_(cuts)
        for x in outs:
            x.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        want = [torch.full_like(q, 3.0) for _ in range(3)]
        step(want)
        assert all(R.same(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
def test_starts_that_do_not_ascend(ctx, cache_type):
    """Every output is what slots and rows can give, whosever a row is."""
    from provekv_amd.paged import PagedKVCache, attend_prompts
    seqs, rows = 300, 900
    g = torch.Generator().manual_seed(78)
    cache = PagedKVCache(1, 2, seqs + 1, 64, 64, dtype=cache_type)
    cache.store(*[torch.ones(1, (seqs + 1) * 64, 2, 64, device="cuda")] * 2, words([list(range(seqs + 1))]), (seqs + 1) * 64)
    bad = cache.buf if cache_type == BF16 else cache.scales
    bad[:, seqs] = math.nan if cache_type == BF16 else 255
    wide = torch.full((seqs, 9), seqs, dtype=torch.int32, device="cuda")
    wide[:, 3] = torch.arange(seqs, dtype=torch.int32, device="cuda")
    tables, n = wide[:, 3:4], words([64] * seqs)
    two = torch.full((1, rows, 2, 64), 2.0, dtype=BF16, device="cuda")
    q = torch.ones(rows, 4, 64, dtype=BF16, device="cuda")
    for starts in ([rows] * seqs + [0], [0, rows] * (seqs // 2) + [rows], torch.randint(-9, rows + 9, (seqs + 1,), generator=g).tolist(),
                   torch.randint(-2 ** 31, 2 ** 31 - 1, (seqs + 1,), generator=g).tolist()):
        st = words(starts)
        cache.store(two, two, tables, n, starts=st)
        for back in cache.load(rows, tables, n, starts=st):
            assert ((back == 0) | (back == 1) | (back == 2)).all()
        for most in (None, 2, 50):
            out = cache.attend(0, q, tables, n, starts=st, out=torch.full_like(q, 55.0), max_rows=most)
            assert (((out >= 1) & (out <= 2)) | (out == 55) | (out == 0)).all()
            out = attend_prompts(q, q[:, :2], q[:, :2], st, out=torch.full_like(q, 55.0), max_rows=most)
            assert ((out == 1) | (out == 55)).all()


def test_time_by_the_sequences(ctx):
    """65,536 single tokens and prompts of four rows: single milliseconds.  Counted
    by every workgroup for itself it would be 0.3 s and more."""
    from provekv_amd.paged import PagedKVCache, attend_prompts
    seqs = 1 << 16
    cache = PagedKVCache(1, 1, 64, 16, 64, dtype=BF16)
    cache.buf.normal_()
    tables = torch.randint(0, 64, (seqs, 2), device="cuda", dtype=torch.int32)
    lens, st = words([20] * seqs), torch.arange(seqs + 1, device="cuda", dtype=torch.int32)
    q = torch.randn(seqs, 1, 64, device="cuda").bfloat16()
    x = torch.randn(seqs * 4, 3, 64, device="cuda").bfloat16()
    for call in (lambda: cache.attend(0, q, tables, lens), lambda: cache.attend(0, q, tables, lens, starts=st),
                 lambda: attend_prompts(x[:, :1], x[:, 1:2], x[:, 2:], st * 4), lambda: cache.load(seqs, tables, lens, starts=st)):
        call()
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        assert a.elapsed_time(b) < 100.0

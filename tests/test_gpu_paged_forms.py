"""Forms of paged and packed calls that the documentation allows: one length for
all with starts and windows, operands whose heads or rows are one and the same
memory, a table that all sequences share, a row of queries that is not finite,
calls on two streams at once, 8-bit pages a caller filled with any codes and scales."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
from test_gpu_paged import BF16, F16, F8, KIND_IDS, KINDS, make, running, run, sequences, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,G", [([1, 1, 1], 2), ([2, 0, 1], 20), ([40, 1, 9], 1)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 2)])
def test_one_length_with_starts(ctx, window, sinks, counts, G, cache_type, dtype):
    """Past the table's slots it is taken as they are; below 1 there are none."""
    cache, tables = make(cache_type, 2, 64, 16, [200] * 3, seed=80)
    rows, st = sum(counts), words(running(counts))
    q = torch.randn(rows, 2 * G, 64, generator=torch.Generator().manual_seed(81)).to(dtype)
    spans = P.rows_of(running(counts), 3, rows)
    for n in (1, 77, 200, 208, 10 ** 9):
        lse = torch.full((2 * G, rows), 77.0, device="cuda")
        out = cache.attend(0, q.cuda(), words(tables), n, starts=st, window=window, sinks=sinks, lse=lse)
        lens = [min(n, 16 * len(tables[0]))] * 3
        ref = P.attend(q.double(), sequences(cache, tables, lens), lens, spans, window, sinks, 0.125)
        P.check(out, lse, ref, spans, dtype)
    for n in (0, -5):
        assert not cache.attend(0, q.cuda(), words(tables), n, starts=st).any()
    keys, values = cache.load(rows, words(tables), 77, starts=st, layer=0)
    back = cache.load(rows, words(tables), words([77] * 3), starts=st, layer=0)
    assert R.same(keys, back[0]) and R.same(values, back[1]) and keys.any()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("rows", [3, 60])
def test_memory_that_heads_and_rows_share(ctx, rows, cache_type, dtype):
    """Queries, keys and values expanded over heads or rows; one table for all."""
    from provekv_amd.paged import attend_prompts
    cache, tables = make(cache_type, 2, 64, 16, [90], seed=82)
    g = torch.Generator(device="cuda").manual_seed(83)
    st = words([0, rows - 2, rows - 1, rows])
    t = words(tables)
    for q in (torch.randn(rows, 1, 64, device="cuda", generator=g).to(dtype).expand(rows, 4, 64),
              torch.randn(1, 4, 64, device="cuda", generator=g).to(dtype).expand(rows, 4, 64)):
        a = cache.attend(0, q, t.expand(3, -1), words([90, 40, 7]), starts=st)
        b = cache.attend(0, q.contiguous(), t.expand(3, -1).contiguous(), words([90, 40, 7]), starts=st)
        assert R.same(a, b) and torch.isfinite(a).all() and a.any()
        k = torch.randn(rows, 1, 64, device="cuda", generator=g).to(dtype)
        a = attend_prompts(q, k.expand(rows, 2, 64), k[:, :, :].expand(rows, 2, 64), st)
        b = attend_prompts(q.contiguous(), k.repeat(1, 2, 1), k.repeat(1, 2, 1), st)
        assert R.same(a, b) and a.any()
    one = torch.randn(1, 1, 1, 64, device="cuda", generator=g).to(dtype)
    cache.store(one.expand(1, 3, 2, 64), one.expand(1, 3, 2, 64), t, 90)
    keys, values = cache.load(3, t, 90, dtype=torch.float32)
    want = P.rounded(one, cache_type).expand(1, 3, 2, 64)
    assert R.same(keys.double(), want) and R.same(values.double(), want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,H", [([1, 4, 1], 2), ([70, 1, 33], 2), ([150] * 4, 32)])
def test_queries_that_are_not_finite(ctx, counts, H, cache_type, dtype, bad):
    """One query row's: the others keep their values (few and many rows share its
    workgroup), its own are NaN."""
    lens = [n + 100 for n in counts]
    cache, tables = make(cache_type, H, 64, 16, lens, seed=84)
    rows = sum(counts)
    q = torch.randn(rows, H, 64, generator=torch.Generator().manual_seed(85)).to(dtype).cuda()
    args = words(tables), words(lens), words(running(counts))
    plain = cache.attend(0, q, args[0], args[1], starts=args[2])
    at = counts[0] + 1
    q[at, H - 1, 7] = bad
    out = cache.attend(0, q, args[0], args[1], starts=args[2])
    assert torch.isnan(out[at, H - 1]).all()
    out[at, H - 1] = plain[at, H - 1]
    # computed again with smaller weights, whose sums may round the other way: a rounding of the type apart
    assert ((out.double() - plain.double()).abs() <= 2 * R.HALF[dtype] * plain.double().abs() + 1e-6).all()


def test_two_streams_at_once(ctx):
    """The same call on two streams, each with a workspace of its own."""
    cache, tables = make(BF16, 4, 128, 64, [9000, 300, 2000], seed=86)
    t, n, st = words(tables), words([9000, 300, 2000]), words([0, 1, 60, 61])
    q = [torch.randn(61, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    want = [cache.attend(0, x, t, n, starts=st) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i in range(2):
            outs[i].append(cache.attend(0, q[i], t, n, starts=st, stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(R.same(x, want[i]) for x in outs[i])


def test_every_code_under_every_scale(ctx):
    """Memory of the caller's own: any of the 256 codes and scale bytes, loaded in
    each type; numbers past f32 are infinities, below it are subnormal."""
    from provekv_amd.paged import PagedKVCache
    buf = torch.arange(256, dtype=torch.uint8).view(1, 1, 1, 2, 1, 128).expand(1, 16, 2, 2, 16, 128).contiguous()
    buf[:, :, 1] = buf[:, :, 1].flip(-1)
    scales = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(1, 16, 1, 1, 16, 1).expand(1, 16, 2, 2, 16, 4).contiguous()
    cache = PagedKVCache.over(buf.cuda(), scales.cuda())
    want = P.values(buf, scales)[0].permute(1, 0, 3, 2, 4).reshape(2, 256, 2, 128)
    for dtype in (torch.float32, BF16, F16):
        got = cache.load(256, words([list(range(16))]), 256, layer=0, dtype=dtype)
        for x, y in zip(got, want):
            assert R.same(x, y.float().to(dtype))


@pytest.mark.parametrize("cache_type,dtype", [(F8, BF16), (F8, F16)], ids=["f8-bf16", "f8-f16"])
@pytest.mark.parametrize("counts", [[1, 1], [50, 3]])
def test_codes_and_scales_of_the_callers(ctx, counts, cache_type, dtype):
    """Scales that differ from block to block, some far below what a store gives."""
    lens = [120, 61]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=87)
    g = torch.Generator(device="cuda").manual_seed(88)
    cache.buf.random_(0, 256, generator=g)
    cache.buf[(cache.buf & 127) == 127] = 1
    cache.scales.random_(116, 122, generator=g)
    cache.scales[:, :, :, :, ::5, 0] = 0
    run(cache, dtype, tables, lens, counts, 2)

"""Attention over paged caches (bf16, f16 and 8-bit) and of packed prompts: every
output against a plain 64-bit form within bounds derived from the arithmetic
(live_ref.py, paged_ref.py)."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P

pytestmark = pytest.mark.gpu
BF16, F16, F8 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
KINDS = [(BF16, BF16), (F16, F16), (F8, BF16), (F8, F16)]
KIND_IDS = ["bf16", "f16", "f8-bf16", "f8-f16"]


def words(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def running(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def make(dtype, H, D, page, lens, seed=0, layers=1, shared=0, spare=2, scale=1.0):
    """(cache, tables as lists): pages in no order, the first `shared` slots'
    pages those of all sequences; entries behind a sequence's length name nothing."""
    from provekv_amd.paged import PagedKVCache
    g = torch.Generator().manual_seed(seed)
    need, common = [(n + page - 1) // page for n in lens], shared // page
    pages = common + sum(max(0, n - common) for n in need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    own, tables = order[common:], []
    for n in need:
        mine = order[:min(n, common)] + own[:max(0, n - common)]
        own = own[max(0, n - common):]
        tables.append(mine + [-1] * (max(max(need), 1) - n))
    x = torch.randn(layers, pages, 2, H, page, D, generator=g) * scale
    x[:, :, 0] *= torch.exp(0.4 * torch.randn(H, 1, D, generator=g))
    cache = PagedKVCache(layers, H, pages, page, D, dtype=dtype)
    if dtype == F8:
        everything = words([[i] for i in range(pages)])
        rows = x.permute(2, 0, 1, 4, 3, 5).reshape(2, layers, pages * page, H, D).cuda()
        cache.store(rows[0], rows[1], everything, page)
    else:
        cache.buf.copy_(x)
    return cache, tables


def sequences(cache, tables, lens, layer=0):
    pages = P.values(cache.buf, cache.scales)[layer]
    return [P.gathered(pages, t, n) for t, n in zip(tables, lens)]


def run(cache, dtype, tables, lens, counts, G, layer=0, window=0, sinks=0, scale=None, seed=1, starts=True, before=0,
        behind=0, **kw):
    """One call with every output, checked.  before, behind: rows of nobody."""
    g = torch.Generator().manual_seed(seed)
    H, D = cache.heads, cache.dim
    rows = before + sum(counts) + behind
    st = [before + x for x in running(counts)] if starts else None
    q = torch.randn(rows, H * G, D, generator=g).to(dtype)
    lse = torch.full((H * G, rows), 77.0, device="cuda")
    out = torch.full((rows, H * G, D), 55.0, dtype=dtype, device="cuda")
    got = cache.attend(layer, q.cuda(), words(tables), words(lens), starts=words(st) if starts else None, window=window,
                       sinks=sinks, scale=scale, lse=lse, out=out, **kw)
    assert got is out
    spans = P.rows_of(st, len(lens), rows)
    ref = P.attend(q.double(), sequences(cache, tables, lens, layer), lens, spans, window, sinks,
                   1 / math.sqrt(D) if scale is None else scale)
    P.check(out, lse, ref, spans, dtype, 55.0, 77.0)
    return out


SIZES = [  # rows of each sequence, lengths, group
    ([1], [1], 1), ([1, 1, 1], [1, 15, 16], 1), ([1, 1, 1, 1], [17, 63, 64, 65], 4), ([1, 1], [257, 300], 3),
    ([1], [130], 16), ([1], [99], 17), ([2, 2], [129, 2], 8), ([5, 0, 3], [130, 40, 3], 3), ([16, 1, 7], [64, 16, 90], 1),
    ([33, 2], [90, 33], 1), ([64, 1, 20], [150, 100, 20], 2), ([130, 0, 131], [257, 31, 131], 1),
    ([200, 1, 1], [333, 150, 1], 3),
]


@pytest.mark.parametrize("D,page", [(64, 16), (128, 64), (128, 16), (64, 32)])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,lens,G", SIZES)
def test_sizes(ctx, counts, lens, G, cache_type, dtype, D, page):
    cache, tables = make(cache_type, 2, D, page, lens, seed=sum(lens))
    run(cache, dtype, tables, lens, counts, G)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n,G", [(1, 1), (1, 5), (4, 4), (3, 7), (40, 2)])
def test_even_rows(ctx, n, G, cache_type, dtype):
    """As many rows for each sequence, without starts."""
    lens = [70, 41, 40, 200, n, 123]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=2)
    run(cache, dtype, tables, lens, [n] * 6, G, starts=False)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (65, 4), (100, 64), (1000, 5), (3, 500)])
@pytest.mark.parametrize("counts,G", [([1, 1, 1], 4), ([6, 1, 3], 2), ([90, 1, 30], 1)])
def test_windows(ctx, counts, G, window, sinks, cache_type, dtype):
    lens = [400, 211, 30]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=3)
    run(cache, dtype, tables, lens, counts, G, window=window, sinks=sinks)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts", [[3, 0, 1], [50, 0, 2]])
def test_rows_of_nobody(ctx, counts, cache_type, dtype):
    lens = [80, 5, 60]
    cache, tables = make(cache_type, 2, 128, 32, lens, seed=4)
    run(cache, dtype, tables, lens, counts, 2, before=3, behind=70)
    run(cache, dtype, tables, lens, [0, 0, 0], 2, before=0, behind=5)
    # a new out: 0 there
    q = torch.randn(3 + sum(counts) + 70, 4, 128, device="cuda").to(dtype)
    st = words([3 + x for x in running(counts)])
    torch.full_like(q, 9.0)             # what the next allocation may find
    out = cache.attend(0, q, words(tables), words(lens), starts=st)
    assert not out[:3].any() and not out[3 + sum(counts):].any() and out[3:3 + sum(counts)].any()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,G", [([4, 2, 9], 1), ([40, 100, 70], 2)])
def test_rows_before_the_first_slot(ctx, counts, G, cache_type, dtype):
    """More rows than slots: those in front see nothing and give 0."""
    lens = [1, 0, counts[2] - 1]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=5)
    out = run(cache, dtype, tables, lens, counts, G)
    assert not out[:counts[0] - 1].any() and not out[counts[0]:counts[0] + counts[1]].any()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,G", [([1, 1, 1], 2), ([30, 1, 65], 2)])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_missing_pages(ctx, counts, G, bad, cache_type, dtype):
    """Slots without a page are seen by no row: one in the middle, the first, all."""
    lens = [100, 200, 90]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=6)
    tables[0][2], tables[1][0], tables[1][12] = bad, bad, bad
    tables[2] = [bad] * len(tables[2])
    out = run(cache, dtype, tables, lens, counts, G)
    assert not out[-counts[2]:].any()
    if cache.scales is None:   # .. whatever page 0 holds
        free = [i for i in range(cache.pages) if not any(i in t for t in tables)]
        cache.buf[:, free] = math.nan
        if 0 in free:
            run(cache, dtype, tables, lens, counts, G)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("G,page", [(1, 16), (4, 128)])
def test_long(ctx, G, page, cache_type, dtype):
    """Enough slots that a row's are split over many workgroups, beside short ones."""
    lens = [9001, 300, 4100, 1]
    cache, tables = make(cache_type, 1, 128, page, lens, seed=7)
    run(cache, dtype, tables, lens, [1, 1, 1, 1], G, starts=False)
    run(cache, dtype, tables, lens, [3, 1, 2, 1], G, window=5000, sinks=4)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts", [[24, 1], [3, 16], [70, 2]])
def test_chunks_on_long_caches(ctx, counts, cache_type, dtype):
    lens = [5000, 700]
    cache, tables = make(cache_type, 1, 64, 64, lens, seed=8)
    run(cache, dtype, tables, lens, counts, 2)
    run(cache, dtype, tables, lens, counts, 2, window=3000, sinks=4, scale=0.3)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("seqs", [64, 65, 130])
def test_many_sequences(ctx, seqs, cache_type, dtype):
    lens = [1 + (i * 37) % 190 for i in range(seqs)]
    cache, tables = make(cache_type, 1, 64, 16, lens, seed=9)
    run(cache, dtype, tables, lens, [1] * seqs, 2, starts=False)
    run(cache, dtype, tables, lens, [i % 3 for i in range(seqs)], 1)
    run(cache, dtype, tables, lens, [min(n, 1 + (i % 5) * 9) for i, n in enumerate(lens)], 1)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
def test_shared_pages_and_layers(ctx, cache_type, dtype):
    """Sequences that share a prefix's pages; a layer of several; limits given."""
    lens = [160, 130, 129, 200]
    cache, tables = make(cache_type, 2, 128, 32, lens, seed=10, layers=3, shared=128)
    assert all(t[:4] == tables[0][:4] for t in tables)
    run(cache, dtype, tables, lens, [1, 1, 1, 1], 2, layer=2, starts=False, max_len=200)
    run(cache, dtype, tables, lens, [30, 1, 1, 70], 2, layer=1, max_len=200, max_rows=70, scale=0.05)


def test_one_length(ctx):
    """lens as an int, the call's own size."""
    cache, tables = make(BF16, 2, 64, 16, [200, 200], seed=11)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    for n in (1, 5, 64, 199, 200):
        a = cache.attend(0, q, words(tables), n)
        b = cache.attend(0, q, words(tables), words([n, n]))
        # cut in other ways: each half a step of bf16 from the value, and f32 sums apart
        assert ((a.double() - b.double()).abs() <= 2.0 ** -7 * a.double().abs() + 1e-5).all()


@pytest.mark.parametrize("counts", [[1, 1, 1], [7, 1, 2], [60, 1, 33]])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
def test_strides(ctx, counts, cache_type, dtype):
    """q and out as slices of wider tensors, heads inside rows and the other way."""
    lens = [120, 75, 40]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=12)
    rows, g = sum(counts), torch.Generator().manual_seed(3)
    wide = torch.randn(rows, 9, 64, generator=g).to(dtype).cuda()
    t, n, st = words(tables), words(lens), words(running(counts))
    plain = cache.attend(0, wide[:, 2:6].contiguous(), t, n, starts=st)
    assert R.same(cache.attend(0, wide[:, 2:6], t, n, starts=st), plain)
    turned = wide[:, 2:6].transpose(0, 1).contiguous().transpose(0, 1)
    into = torch.full((4, rows, 64), 5.0, dtype=dtype, device="cuda").transpose(0, 1)
    assert R.same(cache.attend(0, turned, t, n, starts=st, out=into), plain)
    odd = torch.randn(rows, 4, 65, generator=g).to(dtype).cuda()     # rows of 130 bytes: copied
    odd[..., :64] = wide[:, 2:6]
    assert R.same(cache.attend(0, odd[..., :64], t, n, starts=st), plain)
    # the table a slice of a wider one
    wide_t = torch.full((3, t.shape[1] + 5), -7, dtype=torch.int32, device="cuda")
    wide_t[:, 2:2 + t.shape[1]] = t
    assert R.same(cache.attend(0, wide[:, 2:6], wide_t[:, 2:2 + t.shape[1]], n, starts=st), plain)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("counts,G", [([1, 1], 2), ([4, 3], 2), ([70, 41], 1)])
def test_hidden_slots_may_hold_anything(ctx, counts, G, dtype, bad):
    """Slots behind the length, behind a row's own and outside its window: rows
    that do not see them do not change."""
    lens, window, sinks = [260, 150], 40, 3
    cache, tables = make(dtype, 2, 64, 16, lens, seed=13)
    for s in range(2):
        first = lens[s] - counts[s]
        hidden = torch.ones(len(tables[s]) * 16, dtype=torch.bool)
        for i in range(counts[s]):
            hidden[:lens[s]] &= ~R.seen(first + i, lens[s], window, sinks)
        for j in hidden.nonzero().flatten().tolist():
            if tables[s][j // 16] >= 0:
                cache.buf[0, tables[s][j // 16], :, :, j % 16] = bad
    run(cache, dtype, tables, lens, counts, G, window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,G", [([1, 1], 2), ([5, 2], 3), ([80, 33], 1), ([150, 1], 2)])
def test_seen_values_that_are_not_finite(ctx, counts, G, cache_type, dtype, side, bad):
    """One row of the cache is not finite: rows that see it get what the formula
    gives (an infinity among the values stays one), the others keep their values."""
    lens = [200, 90]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=14)
    j = lens[0] - counts[0] // 2 - 1                  # seen by about half of the rows
    page = tables[0][j // 16]
    if cache_type == F8:
        cache.scales[0, page, side, 1, j % 16, 1] = 255          # a block of NaN
    else:
        cache.buf[0, page, side, 1, j % 16, 37] = bad
    g = torch.Generator().manual_seed(4)
    rows, st = sum(counts), running(counts)
    q = torch.randn(rows, 2 * G, 64, generator=g).to(dtype)
    out = cache.attend(0, q.cuda(), words(tables), words(lens), starts=words(st)).cpu().double()
    spans = P.rows_of(st, 2, rows)
    kv = sequences(cache, tables, lens)
    ref = P.attend(q.double(), kv, lens, spans, 0, 0, 0.125)
    if side == 1:
        P.check(out.to(dtype), None, ref, spans, dtype)
        return
    # among the keys: the logit is not finite; rows that do not see the slot are as ever
    clean = torch.ones(rows, 2 * G, dtype=torch.bool)
    clean[max(0, counts[0] - (lens[0] - j)):counts[0], G:] = False
    bound = R.out_bound(ref, dtype)
    err = ((out - ref["out"]).abs() - bound)[clean]
    assert not torch.isnan(err).any() and not (err > 0).any()
    k_is_nan = cache_type == F8 or math.isnan(bad)
    if k_is_nan:
        assert torch.isnan(out[~clean]).all()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts", [[1, 1], [50, 2]])
def test_large_logits_and_values(ctx, counts, cache_type, dtype):
    """Logits in the hundreds, and values near the end of the type."""
    lens = [300, 41]
    cache, tables = make(cache_type, 1, 64, 16, lens, seed=15)
    run(cache, dtype, tables, lens, counts, 2, scale=8.0)
    big = {BF16: 2.0 ** 126, F16: 2.0 ** 14, F8: 2.0 ** 14 if dtype == F16 else 2.0 ** 118}[cache_type]
    if cache_type == F8:
        cache.buf.random_(0, 256)
        cache.buf[(cache.buf & 127) == 127] = 0x7e
        cache.scales[:, :, 0].fill_(110)
        cache.scales[:, :, 1].fill_(127 + int(math.log2(big)) - 8)
    else:
        cache.buf[:, :, 1] = torch.rand(cache.buf[:, :, 1].shape, device="cuda").to(dtype) * big
    run(cache, dtype, tables, lens, counts, 2)


PROMPTS = [([1], 1), ([2, 1, 3], 4), ([17], 3), ([63, 64, 65], 1), ([127, 128, 129], 2), ([300, 5, 0, 77], 3),
           ([31, 257, 1, 1, 1], 16), ([200], 17)]


def prompts(dtype, counts, H, G, D, before=0, behind=0, seed=0, fused=True):
    g = torch.Generator().manual_seed(seed)
    rows = before + sum(counts) + behind
    x = torch.randn(rows, H * (G + 2), D, generator=g).to(dtype)
    q, k, v = x[:, :H * G], x[:, H * G:H * G + H], x[:, H * G + H:]
    d = x.cuda()
    dev = (d[:, :H * G], d[:, H * G:H * G + H], d[:, H * G + H:])
    if not fused:
        dev = tuple(t.contiguous() for t in dev)
    return (q, k, v), dev, [before + y for y in running(counts)]


def run_prompts(dtype, counts, H, G, D, window=0, sinks=0, scale=None, before=0, behind=0, seed=0, fused=True, **kw):
    from provekv_amd.paged import attend_prompts
    (q, k, v), (dq, dk, dv), st = prompts(dtype, counts, H, G, D, before, behind, seed, fused)
    rows = q.shape[0]
    lse = torch.full((H * G, rows), 77.0, device="cuda")
    out = torch.full((rows, H * G, D), 55.0, dtype=dtype, device="cuda")
    got = attend_prompts(dq, dk, dv, words(st), window=window, sinks=sinks, scale=scale, lse=lse, out=out, **kw)
    assert got is out
    spans = P.rows_of(st, len(counts), rows)
    kv = [(k[a:a + m].double().transpose(0, 1), v[a:a + m].double().transpose(0, 1), torch.ones(m, dtype=torch.bool))
          for a, m in spans]
    ref = P.attend(q.double(), kv, counts, spans, window, sinks, 1 / math.sqrt(D) if scale is None else scale)
    P.check(out, lse, ref, spans, dtype, 55.0, 77.0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("counts,G", PROMPTS)
def test_prompts(ctx, counts, G, dtype, D):
    run_prompts(dtype, counts, 2, G, D, fused=G != 4)
    run_prompts(dtype, counts, 1, G, D, before=2, behind=30, max_rows=max(counts))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (65, 4), (100, 64), (1000, 5), (3, 500)])
def test_prompts_windows(ctx, window, sinks, dtype):
    run_prompts(dtype, [230, 40, 301], 2, 2, 64, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_prompts_many(ctx, dtype):
    run_prompts(dtype, [i % 7 * 5 for i in range(150)], 1, 2, 64)
    run_prompts(dtype, [1400, 3], 1, 1, 64, scale=0.5)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_prompts_values_that_are_not_finite(ctx, dtype, bad):
    """A value that is not finite reaches the rows that see it and no others: not
    those before it, not another sequence's, not those whose window has passed it."""
    from provekv_amd.paged import attend_prompts
    counts, G = [100, 150, 30], 2
    for window, j in ((0, 160), (20, 160), (0, 249), (0, 100)):
        (q, k, v), (dq, dk, dv), st = prompts(dtype, counts, 2, G, 64, seed=5)
        v[j, 1, 9], dv[j, 1, 9] = bad, bad
        dv_before = dv.clone()
        out = attend_prompts(dq, dk, dv, words(st), window=window)
        assert R.same(dv, dv_before)
        spans = P.rows_of(st, 3, 280)
        kv = [(k[a:a + m].double().transpose(0, 1), v[a:a + m].double().transpose(0, 1), torch.ones(m, dtype=torch.bool))
              for a, m in spans]
        ref = P.attend(q.double(), kv, counts, spans, window, 0, 0.125)
        P.check(out, None, ref, spans, dtype)
        assert torch.isfinite(out[:j]).all() and not torch.isfinite(out[j, 2:, 9]).any()


def test_words_are_read_on_the_device(ctx):
    """A captured call, replayed with other tables, lengths and starts, against
    the same call made eagerly; both calls of both kinds in one graph."""
    from provekv_amd.paged import attend_prompts
    lens = [300, 200, 150]
    cache, tables = make(F8, 2, 64, 16, lens, seed=16)
    t, n, st = words(tables), words(lens), words([0, 1, 30, 31])
    q = torch.randn(64, 4, 64, device="cuda").bfloat16()
    k, v = (torch.randn(64, 2, 64, device="cuda").bfloat16() for _ in range(2))
    new = torch.randn(2, 1, 64, 2, 64, device="cuda").bfloat16()

    def step(out):
        cache.store(new[0], new[1], t, n, starts=st)
        return (cache.attend(0, q, t, n, starts=st, out=out[0]), attend_prompts(q, k, v, st, out=out[1]),
                cache.attend(0, q[:3], t, n), *cache.load(64, t, n, starts=st))

    outs = [torch.zeros_like(q) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(outs)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(outs)
    for lens, starts in (([300, 200, 150], [0, 1, 30, 31]), ([299, 0, 31], [0, 0, 0, 40]), ([20, 100, 100], [2, 60, 61, 61]),
                         ([7, 199, 2], [0, 3, 4, 64])):
        n.copy_(words(lens))
        st.copy_(words(starts))
        t.copy_(t.flip(0).contiguous() if lens[0] == 20 else t)
        new.normal_()
        for x in outs:
            x.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        want = step([torch.full_like(q, 3.0) for _ in range(2)])
        for a, b in zip(captured, want):
            assert R.same(a, b)


def test_another_stream(ctx):
    from provekv_amd.paged import attend_prompts
    cache, tables = make(BF16, 2, 64, 16, [90, 50], seed=17)
    q = torch.randn(40, 4, 64, device="cuda").bfloat16()
    k, v = (torch.randn(40, 2, 64, device="cuda").bfloat16() for _ in range(2))
    t, n, st = words(tables), words([90, 50]), words([0, 35, 40])
    a, b = cache.attend(0, q, t, n, starts=st), attend_prompts(q, k, v, st)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    c, d = cache.attend(0, q, t, n, starts=st, stream=s), attend_prompts(q, k, v, st, stream=s)
    s.synchronize()
    assert R.same(a, c) and R.same(b, d)
    keys, values = cache.load(40, t, n, starts=st, layer=0, stream=s)
    cache.store(keys, values, t, n, starts=st, layer=0, stream=s)
    s.synchronize()
    assert R.same(cache.attend(0, q, t, n, starts=st), a)


def test_repeated(ctx):
    """The same call gives the same bits."""
    lens = [3000, 500, 900]
    cache, tables = make(F8, 2, 128, 16, lens, seed=18)
    q = torch.randn(300, 8, 128, device="cuda").bfloat16()
    st = words([0, 298, 299, 300])
    a = cache.attend(0, q, words(tables), words(lens), starts=st)
    for _ in range(3):
        assert R.same(cache.attend(0, q, words(tables), words(lens), starts=st), a)


def test_no_rows(ctx):
    from provekv_amd.paged import attend_prompts
    cache, tables = make(BF16, 2, 64, 16, [20], seed=19)
    q = torch.zeros(0, 4, 64, dtype=BF16, device="cuda")
    assert cache.attend(0, q, words(tables), words([20])).shape == q.shape
    assert attend_prompts(q, q[:, :2], q[:, 2:], words([0, 0])).shape == q.shape
    keys, values = cache.load(0, words(tables), words([20]))
    cache.store(keys, values, words(tables), words([20]))


@pytest.mark.parametrize("starts", [[0, 20, 5, 6], [0, 300, 0, 300], [300, 200, 100, 0], [-5, 7, 10 ** 9, 3]])
def test_starts_that_do_not_ascend(ctx, starts):
    """Whose a row is, is not said, but nothing out of a sequence's own slots is
    touched: what follows its table names a page that no call may write or read."""
    from provekv_amd.paged import PagedKVCache, attend_prompts
    lens, page = [320, 320, 320], 16
    cache = PagedKVCache(1, 2, 61 + 1, page, 64, dtype=BF16)
    cache.buf.fill_(1.0)
    cache.buf[:, 61] = math.nan
    wide = torch.full((3, 60), 61, dtype=torch.int32, device="cuda")
    wide[:, :20] = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    tables, n, st = wide[:, :20], words(lens), words(starts)
    rows = torch.full((1, 300, 2, 64), 2.0, dtype=BF16, device="cuda")
    cache.store(rows, rows, tables, n, starts=st)
    torch.cuda.synchronize()
    assert torch.isnan(cache.buf[:, 61]).all() and not torch.isnan(cache.buf[:, :61]).any()
    for back in cache.load(300, tables, n, starts=st):
        assert not torch.isnan(back).any()
    for G in (1, 4):
        q = torch.ones(300, 2 * G, 64, dtype=BF16, device="cuda")
        out = torch.zeros_like(q)
        cache.attend(0, q, tables, n, starts=st, out=out)
        attend_prompts(q, q[:, :2], q[:, :2], st, out=out)
        torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
def test_many_long_sequences(ctx, cache_type, D):
    """Slots enough for the larger number of units; two of the heads against the plain form."""
    from provekv_amd.paged import PagedKVCache
    H, page, G = 16, 128, 2
    lens = [17000, 20000, 16500, 18001, 17777, 19000, 16900, 20000, 18500, 17400, 16800, 19990]     # 217,868
    need = [(n + page - 1) // page for n in lens]
    g = torch.Generator().manual_seed(20)
    order = torch.randperm(sum(need), generator=g).tolist()
    tables = [[order.pop() for _ in range(n)] + [-1] * (max(need) - n) for n in need]
    cache = PagedKVCache(1, H, sum(need), page, D, dtype=cache_type)
    dg = torch.Generator(device="cuda").manual_seed(21)
    if cache_type == F8:
        cache.buf.random_(0, 256, generator=dg)
        cache.buf[(cache.buf & 127) == 127] = 0
        cache.scales.random_(118, 121, generator=dg)
    else:
        cache.buf.normal_(generator=dg)
    q = torch.randn(len(lens), H * G, D, generator=g).to(BF16)
    out = cache.attend(0, q.cuda(), words(tables), words(lens))
    some = [0, 15]
    pages = P.values(cache.buf[:, :, :, some], None if cache_type == BF16 else cache.scales[:, :, :, some])[0]
    kv = [P.gathered(pages, t, n) for t, n in zip(tables, lens)]
    spans = [(i, 1) for i in range(len(lens))]
    rows = [h * G + y for h in some for y in range(G)]
    P.check(out[:, rows], None, P.attend(q[:, rows].double(), kv, lens, spans, 0, 0, 1 / math.sqrt(D)), spans, BF16)

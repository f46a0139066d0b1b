"""Rows into pages and back: every value against the plain rounding, every slot
that no row has as it was."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
from test_gpu_paged import BF16, F16, F8, make, running, words

pytestmark = pytest.mark.gpu
F32 = torch.float32
TYPES = [(c, r) for c in (BF16, F16, F8) for r in (F32, BF16, F16)]
IDS = [f"{c}-{r}".replace("torch.", "") for c, r in TYPES]


def put(cache, rows, tables, lens, spans, layer):
    """What the cache should hold afterwards, f64, and the slots written."""
    want = P.values(cache.buf, cache.scales)
    new = P.rounded(rows, cache.buf.dtype)                       # [2, layers, rows, H, D]
    written = torch.zeros(want.shape[0], want.shape[1], cache.page_size, dtype=torch.bool)
    size = cache.page_size
    for t, n, (a, m) in zip(tables, lens, spans):
        for i in range(m):
            j = n - m + i
            if j < 0 or not 0 <= t[j // size] < cache.pages:
                continue
            for k, lay in enumerate(range(cache.layers) if layer is None else [layer]):
                want[lay, t[j // size], :, :, j % size] = new[:, k, a + i]
                written[lay, t[j // size], j % size] = True
    return want, written


def check(cache, rows, tables, lens, counts, layer=None, starts=True, before=0, behind=0):
    total = before + sum(counts) + behind
    st = [before + x for x in running(counts)] if starts else None
    spans = P.rows_of(st, len(lens), total)
    want, _ = put(cache, rows, tables, lens, spans, layer)
    d = rows.cuda() if layer is None else rows[:, 0].cuda()
    t, n, s = words(tables), words(lens), None if st is None else words(st)
    cache.store(d[0], d[1], t, n, starts=s, layer=layer)
    assert R.same(P.values(cache.buf, cache.scales), want)
    keys, values = cache.load(total, t, n, starts=s, layer=layer, dtype=rows.dtype)
    got = torch.stack((keys, values)).cpu()
    exact = torch.zeros(got.shape, dtype=torch.float64)
    for tab, length, (a, m) in zip(tables, lens, spans):
        for i in range(m):
            j = length - m + i
            if j >= 0 and 0 <= tab[j // cache.page_size] < cache.pages:
                x = want[:, tab[j // cache.page_size], :, :, j % cache.page_size]      # [layers, 2, H, D]
                exact[..., a + i, :, :] = x.transpose(0, 1) if layer is None else x[layer]
    assert R.same(got, exact.to(rows.dtype))


@pytest.mark.parametrize("D,page", [(64, 16), (128, 32)])
@pytest.mark.parametrize("cache_type,dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("counts,lens", [([1], [1]), ([1, 1, 1], [16, 17, 40]), ([5, 0, 33], [20, 3, 33]),
                                         ([40, 16, 1, 15], [70, 16, 9, 31])])
def test_rows(ctx, counts, lens, cache_type, dtype, D, page):
    H, layers = 3, 2
    cache, tables = make(cache_type, H, D, page, lens, seed=1, layers=layers)
    g = torch.Generator().manual_seed(2)
    rows = (torch.randn(2, layers, sum(counts), H, D, generator=g) * 3).to(dtype)
    check(cache, rows, tables, lens, counts)
    rows = torch.randn(2, 1, 4 + sum(counts) + 9, H, D, generator=g).to(dtype)
    check(cache, rows, tables, lens, counts, layer=1, before=4, behind=9)


@pytest.mark.parametrize("cache_type,dtype", TYPES, ids=IDS)
def test_even_rows_and_missing_slots(ctx, cache_type, dtype):
    """Without starts; rows in front of the first slot, and pages that are none."""
    lens = [50, 2, 17, 0]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=3)
    tables[0][2], tables[2][1] = -1, cache.pages
    g = torch.Generator().manual_seed(4)
    check(cache, torch.randn(2, 1, 4 * 20, 2, 64, generator=g).to(dtype), tables, lens, [20] * 4, starts=False)


@pytest.mark.parametrize("seqs", [64, 65, 200])
def test_many_sequences(ctx, seqs):
    lens = [1 + i * 7 % 40 for i in range(seqs)]
    cache, tables = make(F8, 1, 64, 16, lens, seed=5)
    g = torch.Generator().manual_seed(6)
    counts = [min(n, i % 4) for i, n in enumerate(lens)]
    check(cache, torch.randn(2, 1, sum(counts), 1, 64, generator=g), tables, lens, counts)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_every_scale_and_code(ctx, dtype):
    """Blocks at every power of two and on both sides of the borders: of the
    scale (448 steps), between codes, of the type's ends."""
    g = torch.Generator().manual_seed(7)
    lo, hi = {F32: (-149, 127), BF16: (-133, 127), F16: (-24, 15)}[dtype]
    rows = []
    for e in range(lo, hi + 1):
        m = torch.tensor([1.0, 1.5, 1.75, 1.7578125, 1.9375, 1.25])[e % 6]
        x = (torch.rand(32, generator=g) * 2 - 1).double() * 2.0 ** e
        x[0] = m.double() * 2.0 ** e
        rows.append(x)
    grid = P.table8()[:127]
    between = torch.cat((grid, (grid[1:] + grid[:-1]) / 2, torch.zeros(3).double()))   # codes and the places half way
    for e in (0, -3, -20, 90 if dtype != F16 else 6):
        for part in between.split(31):
            x = torch.zeros(32, dtype=torch.float64)
            x[1:1 + len(part)] = part * 2.0 ** e
            x[0] = 448.0 * 2.0 ** e
            rows.append(-x if e else x)
    x = torch.stack(rows)
    x = torch.cat((x, torch.zeros(-len(x) % 4, 32).double())).to(dtype)
    x = x.view(-1, 128)
    n = x.shape[0]
    from provekv_amd.paged import PagedKVCache
    pages = (n + 15) // 16
    cache = PagedKVCache(1, 1, pages, 16, 128, dtype=F8)
    t = [list(range(pages))]
    check(cache, torch.stack((x, -x)).view(2, 1, n, 1, 128), t, [n], [n])
    assert not torch.isnan(P.values(cache.buf, cache.scales)).any()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cache_type,dtype", TYPES, ids=IDS)
def test_not_finite(ctx, cache_type, dtype, bad):
    cache, tables = make(cache_type, 2, 64, 16, [20], seed=8)
    rows = torch.randn(2, 1, 20, 2, 64).to(dtype)
    rows[0, 0, 3, 1, 40], rows[1, 0, 17, 0, 5] = bad, bad
    check(cache, rows, tables, [20], [20])
    rows = torch.full((2, 1, 20, 2, 64), bad).to(dtype)
    check(cache, rows, tables, [20], [20])


def test_f32_past_the_last_scale(ctx):
    """Values past 448 * 2^119 go to it."""
    cache, tables = make(F8, 1, 64, 16, [2], seed=9)
    x = torch.full((2, 1, 2, 1, 64), 3.4e38)
    x[..., ::3] *= -0.9
    check(cache, x, tables, [2], [2])
    assert P.values(cache.buf, cache.scales)[0, tables[0][0], 0, 0, 0].abs().max() == 448.0 * 2.0 ** 119


@pytest.mark.parametrize("cache_type", [BF16, F8])
def test_one_side_and_strides(ctx, cache_type):
    """Keys or values alone; rows out of a contiguous cache [heads, tokens, dim]; odd strides."""
    lens = [33]
    cache, tables = make(cache_type, 3, 64, 16, lens, seed=10)
    other, _ = make(cache_type, 3, 64, 16, lens, seed=10)
    t, n = words(tables), words(lens)
    x = torch.randn(2, 1, 3, 40, 64, device="cuda")                 # [K|V, layers, heads, tokens, dim]
    rows = x.transpose(2, 3)[:, :, 2:35]
    cache.store(rows[0], rows[1], t, n)
    other.store(rows[0].contiguous(), None, t, n)
    assert R.same(cache.buf[:, :, 0], other.buf[:, :, 0]) and not R.same(cache.buf[:, :, 1], other.buf[:, :, 1])
    odd = torch.zeros(1, 33, 3, 65, device="cuda")
    odd[..., :64] = rows[1]
    other.store(None, odd[..., :64], t, n)
    assert R.same(cache.buf, other.buf) and (cache.scales is None or R.same(cache.scales, other.scales))
    other.store(None, None, t, n)
    # keys and values of different strides
    other.buf.zero_()
    other.store(rows[0], rows[1].contiguous(), t, n)
    a, b = cache.load(33, t, n, dtype=torch.float32), other.load(33, t, n, dtype=torch.float32)
    assert R.same(a[0], b[0]) and R.same(a[1], b[1])


def test_a_type_of_its_own(ctx):
    """float8_e4m3fn memory is taken as the codes."""
    from provekv_amd.paged import PagedKVCache
    cache, tables = make(F8, 1, 64, 16, [10], seed=11)
    same = PagedKVCache.over(cache.buf.view(F8), cache.scales)
    a = cache.load(10, words(tables), 10)
    b = same.load(10, words(tables), 10)
    assert R.same(a[0], b[0]) and R.same(a[1], b[1])

"""Words of a paged call that name nothing, or do not ascend: what no call may
read is NaN, and every output is looked at."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
from test_gpu_paged import BF16, F8, KIND_IDS, KINDS, make, running, sequences, words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [2, 32])
@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
@pytest.mark.parametrize("starts", [[0, 20, 5, 6], [0, 300, 0, 300], [300, 200, 100, 0], [-5, 7, 10 ** 9, 3], [280, 290, 4, 200],
                                    [0, -1, 2 ** 31 - 1, -2 ** 31]])
def test_starts_that_do_not_ascend(ctx, starts, cache_type, heads):
    """Slots hold 1 and stored rows are 2, so a row of a sequence is between them,
    whichever sequence's it is; any other keeps what it was.  Behind each
    sequence's part of the table, and behind its length, stands a page of NaN."""
    from provekv_amd.paged import PagedKVCache, attend_prompts
    lens, page, rows = [320, 320, 304], 16, 300
    cache = PagedKVCache(1, heads, 62, page, 64, dtype=cache_type)
    cache.store(*[torch.ones(1, 62 * page, heads, 64, device="cuda")] * 2, words([list(range(62))]), 62 * page)
    bad = cache.buf if cache_type == BF16 else cache.scales
    bad[:, 61] = math.nan if cache_type == BF16 else 255
    before = P.values(cache.buf[:, 61], None if cache.scales is None else cache.scales[:, 61])
    wide = torch.full((3, 60), 61, dtype=torch.int32, device="cuda")
    wide[:, :20] = torch.arange(60, dtype=torch.int32, device="cuda").view(3, 20)
    wide[2, 19] = 61
    tables, n, st = wide[:, :20], words(lens), words(starts)
    two = torch.full((1, rows, heads, 64), 2.0, dtype=BF16, device="cuda")
    cache.store(two, two, tables, n, starts=st)
    now = P.values(cache.buf, cache.scales)
    assert R.same(now[:, 61], before) and ((now[:, :61] == 1) | (now[:, :61] == 2)).all()
    for back in cache.load(rows, tables, n, starts=st):
        assert ((back == 0) | (back == 1) | (back == 2)).all()
    for G in (1, 4):
        q = torch.ones(rows, heads * G, 64, dtype=BF16, device="cuda")
        for out in (cache.attend(0, q, tables, n, starts=st, out=torch.full_like(q, 55.0)),
                    cache.attend(0, q, tables, n, starts=st, out=torch.full_like(q, 55.0), max_rows=9)):
            assert (((out >= 1) & (out <= 2)) | (out == 55) | (out == 0)).all()
        for most in (None, 9):
            out = attend_prompts(q, q[:, :heads], q[:, :heads], st, out=torch.full_like(q, 55.0), max_rows=most)
            assert ((out == 1) | (out == 55)).all()
    assert R.same(P.values(cache.buf, cache.scales), now)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,G", [([1, 1, 1], 2), ([1, 1, 1], 20), ([30, 1, 65], 2)])
@pytest.mark.parametrize("gone", [-1, 10 ** 6, -2 ** 31, 2 ** 31 - 1])
def test_missing_pages_whatever_page_0_holds(ctx, counts, G, gone, cache_type, dtype):
    """What stands in for a missing page is not a number."""
    lens = [100, 200, 90]
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=60, spare=3)
    free = [i for i in range(cache.pages) if not any(i in t for t in tables)]
    if 0 not in free:                                     # page 0 moves
        for x in (cache.buf, cache.scales):
            if x is not None:
                x[:, free[0]] = x[:, 0]
        tables = [[free[0] if i == 0 else i for i in t] for t in tables]
    (cache.buf if cache_type != F8 else cache.scales)[:, 0] = math.nan if cache_type != F8 else 255
    tables[0][2], tables[1][0], tables[1][12] = gone, gone, gone
    tables[2] = [gone] * len(tables[2])
    g = torch.Generator().manual_seed(61)
    rows, st = sum(counts), running(counts)
    q = torch.randn(rows, 2 * G, 64, generator=g).to(dtype)
    lse = torch.full((2 * G, rows), 77.0, device="cuda")
    out = cache.attend(0, q.cuda(), words(tables), words(lens), starts=words(st), lse=lse)
    spans = P.rows_of(st, 3, rows)
    ref = P.attend(q.double(), sequences(cache, tables, lens), lens, spans, 0, 0, 0.125)
    P.check(out, lse, ref, spans, dtype)
    assert not out[-counts[2]:].any()
    keys, values = cache.load(lens[0], words(tables[:1]), words(lens[:1]), layer=0)
    for x in (keys, values):
        assert torch.isfinite(x).all() and not x[32:48].any() and x[48:].any()

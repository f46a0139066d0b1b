"""Calls whose sequences have more rows than max_rows says (a captured step that
is replayed with longer chunks): the rows up to it are computed at their own
slots, those past it are nobody's."""
import math

import pytest
import torch

import paged_ref as P
from test_gpu_paged import BF16, F16, F8, KIND_IDS, KINDS, make, prompts, running, sequences, words

pytestmark = pytest.mark.gpu

CUT = [  # rows of each sequence, lengths, group, max_rows
    ([5, 1, 3], [70, 40, 33], 1, 2), ([9, 0, 2], [200, 5, 90], 4, 4), ([40, 1, 70], [130, 20, 75], 2, 33),
    ([30, 2, 1], [25, 90, 1], 1, 20), ([300, 1, 150], [700, 300, 200], 2, 130), ([3, 4], [1, 4], 1, 2),
]


def cut(spans, most):
    return [(a, min(m, most)) for a, m in spans]


@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 3)])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,lens,G,most", CUT)
def test_rows_past_the_limit(ctx, counts, lens, G, most, cache_type, dtype, window, sinks):
    """Row i of n stands at slot len - n + i whether or not all n are computed."""
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=30)
    g = torch.Generator().manual_seed(31)
    rows = 2 + sum(counts) + 3
    st = [2 + x for x in running(counts)]
    q = torch.randn(rows, 2 * G, 64, generator=g).to(dtype)
    lse = torch.full((2 * G, rows), 77.0, device="cuda")
    out = torch.full((rows, 2 * G, 64), 55.0, dtype=dtype, device="cuda")
    cache.attend(0, q.cuda(), words(tables), words(lens), starts=words(st), window=window, sinks=sinks, lse=lse, out=out,
                 max_rows=most)
    spans = P.rows_of(st, len(lens), rows)
    ref = P.attend(q.double(), sequences(cache, tables, lens), lens, spans, window, sinks, 0.125)
    P.check(out, lse, ref, cut(spans, most), dtype, 55.0, 77.0)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_prompt_rows_past_the_limit(ctx, window, sinks, dtype):
    from provekv_amd.paged import attend_prompts
    counts, most = [100, 3, 150], 70
    (q, k, v), (dq, dk, dv), st = prompts(dtype, counts, 2, 2, 64, before=1, behind=2, seed=32)
    lse = torch.full((4, q.shape[0]), 77.0, device="cuda")
    out = torch.full_like(dq, 55.0, memory_format=torch.contiguous_format)
    attend_prompts(dq, dk, dv, words(st), window=window, sinks=sinks, lse=lse, out=out, max_rows=most)
    spans = P.rows_of(st, 3, q.shape[0])
    kv = [(k[a:a + m].double().transpose(0, 1), v[a:a + m].double().transpose(0, 1), torch.ones(m, dtype=torch.bool))
          for a, m in spans]
    ref = P.attend(q.double(), kv, counts, spans, window, sinks, 1 / math.sqrt(64))
    P.check(out, lse, ref, cut(spans, most), dtype, 55.0, 77.0)


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("counts,lens,G,most", CUT)
def test_new_outputs_are_0_past_the_limit(ctx, counts, lens, G, most, cache_type, dtype):
    """In a new out, whatever its memory held: as the rows of nobody."""
    from provekv_amd.paged import attend_prompts
    cache, tables = make(cache_type, 2, 64, 16, lens, seed=33)
    rows = 2 + sum(counts) + 3
    st = [2 + x for x in running(counts)]
    q = torch.randn(rows, 2 * G, 64, device="cuda").to(dtype)
    past = torch.ones(rows, dtype=torch.bool)
    for a, m in cut(P.rows_of(st, len(lens), rows), most):
        past[a:a + m] = False

    def new(call):
        torch.full_like(q, 9.0)             # what the next allocation may find
        return call()

    for out in (new(lambda: cache.attend(0, q, words(tables), words(lens), starts=words(st), max_rows=most)),
                new(lambda: attend_prompts(q, q[:, :2], q[:, :2], words(st), max_rows=most))):
        assert not out[past].any() and out[~past].any()


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
def test_many_sequences_past_the_limit(ctx, dtype):
    """More sequences than a wave has lanes, every third of them too long."""
    from provekv_amd.paged import attend_prompts
    counts = [7 if i % 3 else 40 for i in range(200)]
    (q, k, v), (dq, dk, dv), st = prompts(dtype, counts, 1, 2, 64, before=3, behind=5, seed=34)
    torch.full((q.shape[0], 2, 64), 9.0, dtype=dtype, device="cuda")
    out = attend_prompts(dq, dk, dv, words(st), max_rows=11)
    want = torch.zeros_like(out)
    attend_prompts(dq, dk, dv, words(st), max_rows=11, out=want)
    assert torch.equal(out, want) and not out[3 + 11:3 + 40].any() and out[3 + 40].any()


@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
def test_as_many_shares_as_there_can_be(ctx, cache_type):
    """One sequence and head cut into 1,024 shares, every value the largest of its
    type and every weight the same: no sum on the way passes the end of f32."""
    from provekv_amd.paged import PagedKVCache
    page, slots = 65536, 97 * 1024 * 32
    cache = PagedKVCache(1, 1, slots // page + 1, page, 64, dtype=cache_type)
    if cache_type == F8:
        cache.buf[:, :, 1] = 0x7e
        cache.scales[:, :, 1] = 246
        most = 448.0 * 2.0 ** 119
    else:
        most = torch.finfo(BF16).max
        cache.buf[:, :, 1] = most
    q = torch.ones(1, 2, 64, dtype=BF16, device="cuda")
    out = cache.attend(0, q, words([list(range(cache.pages))]), slots)
    # sums of f32 are off by less than half a step of bf16 here
    assert (out.double() == most).all()

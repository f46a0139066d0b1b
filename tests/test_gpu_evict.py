"""Eviction by accumulated attention weight: kept slots, moved rows and weights, exactly."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
KINDS = [torch.float32, torch.bfloat16, torch.float16, "fp4"]
IDS = ["f32", "bf16", "f16", "fp4"]


def make(kind, C, L, H, T, D, seed=0):
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    g = torch.Generator().manual_seed(seed)
    if kind == "fp4":
        return FourBitKVCache.over(
            torch.randint(0, 256, (C, L, 2, H, T, D // 2), generator=g).to(torch.uint8).cuda(),
            torch.randint(100, 140, (C, L, 2, H, T, D // 32), generator=g).to(torch.uint8).cuda())
    return DeviceKVCache.over(torch.randn(C, L, 2, H, T, D, generator=g).to(kind).cuda())


def parts(cache):
    return [cache.codes, cache.scales] if hasattr(cache, "codes") else [cache.buf]


def empty_like(cache, tokens):
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    if hasattr(cache, "codes"):
        return FourBitKVCache(cache.layers, cache.heads, tokens, cache.dim, copies=cache.copies)
    return DeviceKVCache(cache.layers, cache.heads, tokens, cache.dim, dtype=cache.buf.dtype, copies=cache.copies)


def check(cache, w, lens, budget, sinks, recent, in_place, extra=0):
    C, L, H, T = w.shape
    before = [p.clone() for p in parts(cache)]
    into = None if in_place else empty_like(cache, min(budget, T) + extra)
    d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dw = w.cuda()
    kept, new, packed = cache.evict(d_lens, dw, budget, sinks=sinks, recent=recent, into=into)
    target = cache if in_place else into
    assert new.tolist() == [min(max(0, min(n, T)), budget) for n in lens] and d_lens.tolist() == lens
    if in_place:
        assert packed is dw
    else:
        for a, b in zip(parts(cache), before):
            assert R.same(a, b)
        assert R.same(dw.cpu().view(torch.int32), w.view(torch.int32))
    want = [p.clone() if in_place else torch.zeros_like(t) for p, t in zip(before, parts(target))]
    want_w = torch.zeros(packed.shape)
    for c in range(C):
        for l in range(L):
            for h in range(H):
                at = R.evict(w[c, l, h], max(0, min(lens[c], T)), budget, sinks, recent)
                assert kept[c, l, h].tolist() == at + [-1] * (budget - len(at)), (c, l, h)
                want_w[c, l, h, :len(at)] = w[c, l, h][at]
                for t, b in zip(want, before):
                    t[c, l, :, h, :len(at)] = b[c, l, :, h][:, at]
    for a, b in zip(parts(target), want):
        assert R.same(a, b)
    assert R.same(packed.cpu().view(torch.int32), want_w.view(torch.int32))


def weights(C, L, H, T, seed, coarse):
    w = torch.rand(C, L, H, T, generator=torch.Generator().manual_seed(seed)) ** 6 * 50
    return torch.floor(w) if coarse else w


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
@pytest.mark.parametrize("T,budget,sinks,recent,coarse", [
    (1, 1, 0, 0, False), (50, 1, 0, 0, True), (50, 50, 3, 9, False), (50, 20, 4, 16, False), (300, 131, 4, 30, True),
    (1500, 700, 0, 0, True), (1500, 1499, 1, 1, False), (2500, 64, 64, 0, False), (2500, 1100, 0, 1024, True)])
def test_evict(ctx, T, budget, sinks, recent, coarse, in_place, D, kind):
    cache = make(kind, 3, 2, 2, T, D, seed=T)
    lens = [T, max(1, T - T // 3), min(budget, T) // 2]
    check(cache, weights(3, 2, 2, T, T + budget, coarse), lens, budget, sinks, recent, in_place, extra=T % 3)


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
def test_odd_heads_and_slots(ctx, in_place, D, kind):
    check(make(kind, 2, 3, 3, 77, D, seed=9), weights(2, 3, 3, 77, 4, True), [77, 60], 31, 1, 3, in_place)


@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
def test_weights_of_every_kind(ctx, in_place):
    """Zeros of both signs, equal, negative, subnormal, infinite and NaN weights."""
    T = 600
    w = torch.tensor([0.0, -0.0, 1.0, -1.0, 1e-42, -1e-42, math.inf, -math.inf, math.nan, 3e38])[
        torch.randint(0, 10, (2, 1, 3, T), generator=torch.Generator().manual_seed(5))]
    w = torch.where(torch.isnan(w), torch.tensor(math.nan), w)
    for budget in (30, 299, 420):
        check(make(torch.bfloat16, 2, 1, 3, T, 64, seed=6), w.clone(), [600, 431], budget, 2, 3, in_place)
    nan = w.clone()
    nan[1, 0, 0] = math.nan
    nan[1, 0, 1].view(torch.int32).fill_(-1)       # a NaN with the sign bit
    check(make(torch.bfloat16, 2, 1, 3, T, 64, seed=6), nan, [600, 600], 200, 0, 5, in_place)


def test_out_of_range_lengths(ctx):
    check(make(torch.float32, 3, 1, 2, 40, 64), weights(3, 1, 2, 40, 1, False), [-7, 2 ** 31 - 1, 0], 10, 1, 2, True)


def test_one_layer(ctx):
    cache = make(torch.bfloat16, 2, 3, 2, 100, 64, seed=8)
    before = cache.buf.clone()
    w = weights(2, 1, 2, 100, 3, False)[:, 0].cuda()
    w0 = w.cpu()
    kept, new, packed = cache.evict(90, w, 40, sinks=2, recent=10, layer=1)
    assert kept.shape == (2, 2, 40) and new.tolist() == [40, 40] and packed is w
    assert R.same(cache.buf[:, [0, 2]], before[:, [0, 2]])
    for c in range(2):
        for h in range(2):
            at = R.evict(w0[c, h], 90, 40, 2, 10)
            assert kept[c, h].tolist() == at
            assert R.same(cache.buf[c, 1, :, h, :40], before[c, 1, :, h][:, at])


def test_captured(ctx):
    """Replays with new weights and lengths, into another cache."""
    cache = make(torch.bfloat16, 2, 1, 2, 500, 64, seed=9)
    into = empty_like(cache, 200)
    w = torch.zeros(2, 1, 2, 500, device="cuda")
    lens = torch.tensor([500, 450], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.evict(lens, w, 200, sinks=1, recent=50, into=into)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, new, packed = cache.evict(lens, w, 200, sinks=1, recent=50, into=into)
    for k in range(3):
        w.copy_(weights(2, 1, 2, 500, 40 + k, k == 1))
        lens.copy_(torch.tensor([500 - k, 150 + 100 * k], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        other = empty_like(cache, 200)
        kept2, new2, packed2 = cache.evict(lens, w, 200, sinks=1, recent=50, into=other)
        assert R.same(kept, kept2) and R.same(new, new2) and R.same(packed, packed2)
        for c in range(2):
            n = int(new[c])
            assert R.same(into.buf[c, :, :, :, :n], other.buf[c, :, :, :, :n])

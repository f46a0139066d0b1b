"""Eviction: caches longer than the selection holds in registers (32,768 slots),
and the filled length that a cache remembers."""
import pytest
import torch

from test_gpu_evict import IDS, KINDS, check, make, weights

pytestmark = pytest.mark.gpu


def test_filled_length(ctx):
    """In place the cache has at most the budget; another cache keeps the longer of the two."""
    for into_self in (False, True):
        cache = make(torch.bfloat16, 1, 2, 2, 100, 64)
        cache.mark_filled(90)
        cache.evict(90, weights(1, 2, 2, 100, 1, False).cuda(), 40, into=cache if into_self else None)
        assert cache.seq_len() == 40
    cache, other = make(torch.bfloat16, 1, 2, 2, 100, 64), make(torch.bfloat16, 1, 2, 2, 60, 64)
    cache.mark_filled(90)
    for filled, want in ((0, 40), (55, 55)):
        other.mark_filled(filled)
        cache.evict(90, weights(1, 2, 2, 100, 1, False).cuda(), 40, into=other)
        assert cache.seq_len() == 90 and other.seq_len() == want


@pytest.mark.parametrize("kind", KINDS, ids=IDS)
@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
@pytest.mark.parametrize("T,budget,sinks,recent,coarse", [
    (32769, 1, 0, 0, False), (32769, 32768, 4, 1000, True), (40000, 1025, 4, 1000, True), (70001, 3000, 4, 2996, False),
    (70001, 5000, 0, 0, True), (70001, 40000, 7, 20000, False), (70001, 69999, 2, 1, True)])
def test_long(ctx, T, budget, sinks, recent, coarse, in_place, kind):
    """One copy past the registers, one within them, in one launch."""
    lens = [T, min(T, 32768) - 5]
    check(make(kind, 2, 1, 2, T, 64, seed=T), weights(2, 1, 2, T, budget, coarse), lens, budget, sinks, recent, in_place,
          extra=3)


@pytest.mark.parametrize("in_place", [True, False], ids=["in-place", "into"])
def test_long_weights_of_every_kind(ctx, in_place):
    """Equal, infinite and NaN weights past the registers, and a length at each side of the step to them."""
    T = 33000
    w = torch.tensor([0.0, -0.0, 1.0, -1.0, 1e-42, float("inf"), -float("inf"), float("nan"), 3e38])[
        torch.randint(0, 9, (3, 1, 2, T), generator=torch.Generator().manual_seed(5))]
    w = torch.where(torch.isnan(w), torch.tensor(float("nan")), w)
    w[0, 0, 0] = float("nan")
    for budget in (30, 15000):
        check(make(torch.bfloat16, 3, 1, 2, T, 64, seed=6), w.clone(), [T, 32768, 32769], budget, 2, 3, in_place)


def test_long_captured(ctx):
    """Replays in place, from the same start, with lengths of both kinds."""
    cache = make(torch.bfloat16, 1, 1, 2, 50000, 64, seed=9)
    first = cache.buf.clone()
    w = torch.zeros(1, 1, 2, 50000, device="cuda")
    lens = torch.tensor([50000], dtype=torch.int32, device="cuda")
    cache.evict(lens, w.clone(), 4000, sinks=1, recent=50)      # before the capture: the library's first call
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kept, new, packed = cache.evict(lens, w, 4000, sinks=1, recent=50)
    for k, n in enumerate((50000, 30000, 41234, 3999)):
        start = weights(1, 1, 2, 50000, 60 + k, k == 1).cuda()
        runs = []
        for call in (g.replay, None):
            cache.buf.copy_(first)
            w.copy_(start)
            lens.fill_(n)
            if call:
                call()
                out = kept, new, packed
            else:
                out = cache.evict(lens, w, 4000, sinks=1, recent=50)
            torch.cuda.synchronize()
            runs.append([x.cpu().clone() for x in (*out, cache.buf)])
        for a, b in zip(*runs):
            assert torch.equal(a, b)

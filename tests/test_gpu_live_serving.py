"""The live-cache operators as a serving loop uses them: the two-tier plan
rehydrates every agent's cache, prompts and tokens attend to it, a 4-bit copy
serves the same tokens, the accumulated weights shorten both, and decoding goes
on; the same steps replayed from a captured graph."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
LAYERS, HEADS, GROUP, D, PREFIX, AGENTS = 2, 2, 3, 64, 90, [20, 20, 20]
ROOM = 40                                   # slots for the tokens to come


def rehydrated(ctx):
    """One cache per agent, each holding the shared prefix and every agent's tokens."""
    from provekv_amd import synth
    from provekv_amd.pool import DeviceKVCache, TwoTierPlan
    plan = TwoTierPlan(ctx, LAYERS, HEADS, D, PREFIX, AGENTS)
    corpus = synth.corpus_tokens(5, LAYERS, HEADS, plan.tokens, D)
    bufs = plan.alloc()
    plan.encode(torch.from_numpy(corpus.reshape(-1)).cuda(), bufs)
    cache = DeviceKVCache(LAYERS, HEADS, plan.tokens + ROOM, D, dtype=torch.bfloat16, copies=len(AGENTS))
    plan.rehydrate(bufs, cache)
    plan.check_rehydrate(bufs)
    return cache, plan.tokens


def check(cache, values, layer, q, lens, out, window, sinks):
    k, v = values
    n = q.shape[1]
    ref = R.attend(q.cpu().double(), k[:, layer], v[:, layer], lens, [n] * len(lens), window, sinks, 1 / math.sqrt(D))
    err = (out.cpu().double() - ref["out"]).abs() - R.out_bound(ref, torch.bfloat16)
    assert not (err > 0).any() and not torch.isnan(err).any(), float(err.max())
    return ref["weights"]


def values_of(cache):
    full = R.fp4_values(cache.codes, cache.scales) if hasattr(cache, "codes") else cache.buf.cpu().double()
    return full[:, :, 0], full[:, :, 1]


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "4-bit"])
def test_prompt_tokens_eviction(ctx, four):
    from provekv_amd.pool import FourBitKVCache
    cache, n = rehydrated(ctx)
    g = torch.Generator().manual_seed(6)
    C = len(AGENTS)
    if four:
        small = FourBitKVCache(LAYERS, HEADS, cache.tokens, D, copies=C)
        small.store(cache.buf[:, :, 0, :, :n], cache.buf[:, :, 1, :, :n], 0)
        assert R.same(R.fp4_values(small.codes, small.scales)[:, :, 0, :, :n], R.fp4_round(cache.buf[:, :, 0, :, :n]))
        cache = small
    weights = torch.zeros(C, LAYERS, HEADS, cache.tokens, device="cuda")
    total = torch.zeros(C, LAYERS, HEADS, cache.tokens, dtype=torch.float64)
    window, sinks = 64, 4

    def attend(rows, lens):
        lens_d = torch.tensor(lens, dtype=torch.int32, device="cuda")
        for layer in range(LAYERS):
            q = torch.randn(C, rows, HEADS * GROUP, D, generator=g).to(torch.bfloat16).cuda()
            out = cache.attend(layer, q, lens_d, window=window, sinks=sinks, weights=weights[:, layer])
            total[:, layer] += check(cache, values_of(cache), layer, q, lens, out, window, sinks)

    def append(slot):
        kv = torch.randn(2, C, LAYERS, HEADS, 1, D, generator=g).to(torch.bfloat16).cuda()
        if four:
            cache.store(kv[0], kv[1], slot)
        else:
            cache.buf[:, :, 0, :, slot], cache.buf[:, :, 1, :, slot] = kv[0, :, :, :, 0], kv[1, :, :, :, 0]

    attend(50, [n, n - 7, n - 30])          # the agents' prompts
    for step in range(3):
        append(n + step)
        attend(1, [n + step + 1] * C)
    assert ((weights.cpu().double() - total).abs() <= total * 2.0 ** -10 + 1e-6).all()
    before = values_of(cache)
    lens, w0 = [n + 3] * C, weights.cpu()
    kept, new, packed = cache.evict(torch.tensor(lens, dtype=torch.int32, device="cuda"), weights, 60, sinks=sinks, recent=20)
    assert new.tolist() == [60] * C and packed is weights
    after = values_of(cache)
    for c in range(C):
        for layer in range(LAYERS):
            for h in range(HEADS):
                at = R.evict(w0[c, layer, h], n + 3, 60, sinks, 20)
                assert kept[c, layer, h].tolist() == at
                for a, b in zip(after, before):
                    assert R.same(a[c, layer, h, :60], b[c, layer, h, at])
    total = packed.cpu().double()
    for step in range(3):
        append(60 + step)
        attend(1, [60 + step + 1] * C)


def test_captured_step(ctx):
    """Store, attention of every layer and eviction in one graph, replayed with
    other tokens and lengths, against the same calls made eagerly."""
    from provekv_amd.pool import FourBitKVCache
    C, T = 2, 400
    g = torch.Generator().manual_seed(7)

    def fresh():
        cache = FourBitKVCache(LAYERS, HEADS, T, D, copies=C)
        x = torch.randn(2, C, LAYERS, HEADS, T, D, generator=torch.Generator().manual_seed(8)).cuda()
        cache.store(x[0], x[1], 0)
        return cache, FourBitKVCache(LAYERS, HEADS, 150, D, copies=C), torch.zeros(C, LAYERS, HEADS, T, device="cuda")

    k, v = (torch.zeros(C, LAYERS, HEADS, 1, D, device="cuda") for _ in range(2))
    q = torch.zeros(LAYERS, C, 1, HEADS * GROUP, D, device="cuda")
    first, lens = (torch.zeros(C, dtype=torch.int32, device="cuda") for _ in range(2))

    def step(cache, into, weights):
        cache.store(k, v, first)
        outs = [cache.attend(layer, q[layer], lens, window=100, sinks=4, weights=weights[:, layer])
                for layer in range(LAYERS)]
        return outs, cache.evict(lens, weights, 150, sinks=4, recent=50, into=into)

    eager, captured = fresh(), fresh()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*fresh())
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*captured)
    captured[2].zero_()
    for n in (300, 301, 399, 150):
        x = torch.randn(2, C, LAYERS, HEADS, 1, D, generator=g)
        k.copy_(x[0])
        v.copy_(x[1])
        q.copy_(torch.randn(q.shape, generator=g))
        first.fill_(n - 1)
        lens.copy_(torch.tensor([n, n - 40], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step(*eager)
        for a, b in zip(got[0], want[0]):
            assert R.same(a, b)
        for a, b in zip(got[1], want[1]):
            assert R.same(a, b)
        assert R.same(captured[2], eager[2]) and R.same(captured[0].codes, eager[0].codes)
        for c, m in enumerate(want[1][1].tolist()):
            assert R.same(captured[1].codes[c, :, :, :, :m], eager[1].codes[c, :, :, :, :m])


@pytest.mark.parametrize("layer", [0, 1])
def test_memory_exchanged(ctx, layer):
    """A cache whose tensors are exchanged for others of the same shape is read where they are now."""
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    g = torch.Generator(device="cuda").manual_seed(9)
    q = torch.randn(2, 3, 4, D, device="cuda", generator=g).bfloat16()
    cache, four = DeviceKVCache(2, 2, 70, D, dtype=torch.bfloat16, copies=2), FourBitKVCache(2, 2, 70, D, copies=2)
    for step in range(2):
        buf = torch.randn(2, 2, 2, 2, 70, D, device="cuda", generator=g).bfloat16()
        cache.buf = buf
        four.codes, four.scales = torch.zeros_like(four.codes), torch.zeros_like(four.scales)
        four.store(buf[:, :, 0], buf[:, :, 1], 0)
        for one in (cache, four):
            k, v = values_of(one)
            weights = torch.zeros(2, 2, 70, device="cuda")
            check(one, (k, v), layer, q, [70, 70], one.attend(layer, q, 70, weights=weights), 0, 0)
            into = type(one)(2, 2, 20, D, copies=2) if one is four else type(one)(2, 2, 20, D, dtype=buf.dtype, copies=2)
            kept, _, _ = one.evict(70, weights, 20, layer=layer, into=into)
            at = kept.cpu().long()[..., None].expand(-1, -1, -1, D)
            assert R.same(values_of(into)[0][:, layer], k[:, layer].gather(2, at))

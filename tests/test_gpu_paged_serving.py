"""Paged caches as a serving loop uses them: the two-tier plan rehydrates a
shared prefix, its rows go into pages that every sequence names, prompts attend
to themselves and are stored, later chunks and tokens attend to prefix, prompt
and each other; the decode step captured, at two batch sizes in turn; pools and
packed rows past 32 bits."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
from test_gpu_paged import BF16, F8, running, words

pytestmark = pytest.mark.gpu
LAYERS, HEADS, GROUP, D, PREFIX, PAGE = 2, 2, 3, 64, 96, 16
SCALE = 1 / math.sqrt(D)


class Serving:
    """Sequences of one pool: rows kept on the CPU as the pages hold them."""

    def __init__(self, ctx, cache_type, room):
        from provekv_amd import synth
        from provekv_amd.pool import DeviceKVCache, PagedKVCache, TwoTierPlan
        plan = TwoTierPlan(ctx, LAYERS, HEADS, D, PREFIX, [8])
        corpus = synth.corpus_tokens(5, LAYERS, HEADS, plan.tokens, D)
        bufs = plan.alloc()
        plan.encode(torch.from_numpy(corpus.reshape(-1)).cuda(), bufs)
        flat = DeviceKVCache(LAYERS, HEADS, plan.tokens, D, dtype=BF16, copies=1)
        plan.rehydrate(bufs, flat)
        plan.check_rehydrate(bufs)
        self.type, self.g = cache_type, torch.Generator().manual_seed(6)
        self.pages = PagedKVCache(LAYERS, HEADS, PREFIX // PAGE + 3 * room, PAGE, D, dtype=cache_type)
        self.free = torch.randperm(self.pages.pages, generator=self.g).tolist()
        self.prefix = [self.free.pop() for _ in range(PREFIX // PAGE)]
        # [K|V][layers, tokens, heads, dim]: views of the rehydrated cache
        both = [flat.buf[0, :, side, :, :PREFIX].transpose(1, 2) for side in range(2)]
        self.pages.store(*both, words([self.prefix]), PREFIX)
        self.tables = [list(self.prefix) for _ in range(3)]
        self.rows = [[P.rounded(x, cache_type) for x in both] for _ in range(3)]

    def grow(self, new):
        """Pages for `new` more rows of each sequence, and the words of the calls."""
        lens = [self.rows[s][0].shape[1] + n for s, n in enumerate(new)]
        for s, n in enumerate(lens):
            while len(self.tables[s]) * PAGE < n:
                self.tables[s].append(self.free.pop())
        most = max(map(len, self.tables))
        return words([t + [-1] * (most - len(t)) for t in self.tables]), lens, running(new)

    def random(self, rows):
        return [torch.randn(LAYERS, rows, HEADS, D, generator=self.g).to(BF16) for _ in range(2)]

    def keep(self, kv, starts):
        for s in range(3):
            for side in range(2 if starts[s + 1] > starts[s] else 0):
                own = P.rounded(kv[side][:, starts[s]:starts[s + 1]], self.type)
                self.rows[s][side] = torch.cat((self.rows[s][side], own), 1)

    def check(self, layer, q, out, lens, starts, window, sinks):
        kv = [(k[layer].transpose(0, 1), v[layer].transpose(0, 1), torch.ones(k.shape[1], dtype=torch.bool))
              for k, v in self.rows]
        spans = P.rows_of(starts, 3, q.shape[0])
        P.check(out, None, P.attend(q.double(), kv, lens, spans, window, sinks, SCALE), spans, BF16)

    def step(self, new, window=0, sinks=0):
        """Rows of the sequences into their pages, then attention over all of them."""
        tables, lens, starts = self.grow(new)
        n, st = words(lens), words(starts)
        kv = self.random(starts[-1])
        self.pages.store(kv[0].cuda(), kv[1].cuda(), tables, n, starts=st)
        self.keep(kv, starts)
        for layer in range(LAYERS):
            q = torch.randn(starts[-1], HEADS * GROUP, D, generator=self.g).to(BF16)
            out = self.pages.attend(layer, q.cuda(), tables, n, starts=st, window=window, sinks=sinks)
            self.check(layer, q, out, lens, starts, window, sinks)
        return tables, n


@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
def test_prefix_prompts_chunks_tokens(ctx, cache_type):
    from provekv_amd.pool import attend_prompts
    s = Serving(ctx, cache_type, 20)
    # prompts that see only themselves, the same rows stored behind the prefix
    new = [70, 5, 33]
    tables, lens, starts = s.grow(new)
    st = words(starts)
    kv = s.random(starts[-1])
    for layer in range(LAYERS):
        q = torch.randn(starts[-1], HEADS * GROUP, D, generator=s.g).to(BF16)
        out = attend_prompts(q.cuda(), kv[0][layer].cuda(), kv[1][layer].cuda(), st)
        own = [(kv[0][layer, a:z].double().transpose(0, 1), kv[1][layer, a:z].double().transpose(0, 1),
                torch.ones(z - a, dtype=torch.bool)) for a, z in zip(starts[:-1], starts[1:])]
        spans = P.rows_of(starts, 3, starts[-1])
        P.check(out, None, P.attend(q.double(), own, new, spans, 0, 0, SCALE), spans, BF16)
    s.pages.store(kv[0].cuda(), kv[1].cuda(), tables, words(lens), starts=st)
    s.keep(kv, starts)
    s.step([1, 1, 1])
    s.step([1, 40, 1])                  # a chunk among tokens
    s.step([4, 2, 0], window=64, sinks=4)
    tables, n = s.step([1, 1, 1], window=64, sinks=4)
    # what the pages hold, read back: the last rows of each sequence
    keys, values = s.pages.load(6, tables, n, dtype=torch.float32)
    for i in range(3):
        for got, side in ((keys, 0), (values, 1)):
            assert R.same(got[:, 2 * i:2 * i + 2].double(), s.rows[i][side][:, -2:])
    # the shared pages were written once and are as they were
    keys, values = s.pages.load(PREFIX, words([s.prefix]), PREFIX, dtype=torch.float32)
    assert R.same(keys.double(), s.rows[0][0][:, :PREFIX]) and R.same(values.double(), s.rows[0][1][:, :PREFIX])


@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
def test_two_captured_decode_steps(ctx, cache_type):
    """Decode steps of 4 and of 16 sequences, captured one after the other into
    one memory pool, replayed in turn on growing lengths, with eager calls between."""
    from provekv_amd.pool import PagedKVCache
    g = torch.Generator().manual_seed(9)
    N, room = 16, 40
    caches = [PagedKVCache(LAYERS, HEADS, N * room, PAGE, D, dtype=cache_type) for _ in range(2)]
    tables = words(torch.randperm(N * room, generator=g).view(N, room).tolist())
    first = [torch.randn(LAYERS, N * 500, HEADS, D, generator=g).to(BF16).cuda() for _ in range(2)]
    for c in caches:
        c.store(first[0], first[1], tables, 500)
    q = torch.randn(LAYERS, N, HEADS * GROUP, D, generator=g).to(BF16).cuda()
    new = torch.randn(2, LAYERS, N, HEADS, D, generator=g).to(BF16).cuda()
    lens = words([500] * N)

    def step(cache, n):
        cache.store(new[0][:, :n], new[1][:, :n], tables[:n], lens[:n])
        return [cache.attend(layer, q[layer][:n], tables[:n], lens[:n]) for layer in range(LAYERS)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for n in (4, N):
            step(caches[0], n)
    torch.cuda.current_stream().wait_stream(side)
    step(caches[1], 4)
    step(caches[1], N)
    torch.cuda.synchronize()
    graphs, outs = {}, {}
    for n in (4, N):
        graphs[n] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[n], pool=graphs[4].pool() if n == N else None):
            outs[n] = step(caches[0], n)
    for i in range(6):
        n = (N, 4, 4, N, 4, N)[i]
        lens.copy_(words([min(500 + 23 * i + 7 * s, room * PAGE) for s in range(N)]))
        new.normal_()
        q.normal_()
        graphs[n].replay()
        got = [x.clone() for x in outs[n]]
        torch.cuda.synchronize()
        for a, b in zip(got, step(caches[1], n)):
            assert R.same(a, b)
    assert R.same(caches[0].buf, caches[1].buf)


@pytest.mark.parametrize("cache_type", [BF16, F8], ids=["bf16", "8-bit"])
@pytest.mark.parametrize("counts", [[1, 1], [5, 90]])
def test_pages_past_32_bits(ctx, cache_type, counts):
    """A pool of more than 2^32 elements, its first and last pages used."""
    from provekv_amd.pool import PagedKVCache
    pages = (1 << 21) + 1000                                # of 2,048 elements
    cache = PagedKVCache(1, 1, pages, 16, 64, dtype=cache_type)
    assert cache.buf.numel() > 1 << 32
    g = torch.Generator().manual_seed(10)
    lens, order = [100, 90], [i if j % 2 else pages - 1 - i for j, i in enumerate(torch.randperm(14, generator=g).tolist())]
    tables = words([order[:7], order[7:]])
    kv = torch.randn(2, 1, 190, 1, 64, generator=g).to(BF16)
    st = words([0, 100, 190])
    cache.store(kv[0].cuda(), kv[1].cuda(), tables, words(lens), starts=st)
    back = cache.load(190, tables, words(lens), starts=st, dtype=torch.float32)
    held = [P.rounded(x, cache_type) for x in kv]
    assert all(R.same(a.double(), b) for a, b in zip(back, held))
    rows, starts = sum(counts), running(counts)
    q = torch.randn(rows, 2, 64, generator=g).to(BF16)
    out = cache.attend(0, q.cuda(), tables, words(lens), starts=words(starts))
    own = [(held[0][0, a:z].transpose(0, 1), held[1][0, a:z].transpose(0, 1), torch.ones(z - a, dtype=torch.bool))
           for a, z in ((0, 100), (100, 190))]
    spans = P.rows_of(starts, 2, rows)
    P.check(out, None, P.attend(q.double(), own, lens, spans, 0, 0, SCALE), spans, BF16)


def test_prompt_rows_past_32_bits(ctx):
    """Packed rows 2^22 elements apart: 1,100 of them pass 2^32 elements."""
    from provekv_amd.pool import attend_prompts
    rows, wide, starts = 1100, 1 << 22, [0, 900, 1000, 1100]
    g = torch.Generator().manual_seed(11)
    x = torch.randn(rows, 4, 64, generator=g).to(BF16)
    big = torch.empty(rows * wide, dtype=BF16, device="cuda")
    view = big.view(rows, wide)[:, :256].view(rows, 4, 64)
    view.copy_(x)
    plain = x.cuda()
    got = attend_prompts(view[:, :2], view[:, 2:3], view[:, 3:], words(starts))
    want = attend_prompts(plain[:, :2], plain[:, 2:3], plain[:, 3:], words(starts))
    assert R.same(got, want)
    for s, (a, z) in enumerate(zip(starts[:-1], starts[1:])):
        if s:
            own = [(x[a:z, 2:3].double().transpose(0, 1), x[a:z, 3:].double().transpose(0, 1),
                    torch.ones(z - a, dtype=torch.bool))]
            spans = [(0, z - a)]
            P.check(got[a:z], None, P.attend(x[a:z, :2].double(), own, [z - a], spans, 0, 0, SCALE), spans, BF16)

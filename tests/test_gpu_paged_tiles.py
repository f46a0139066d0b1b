"""Attention of many rows in each of its tiles, over pages and of packed prompts
(the calls of paged_tiles.py, whose tile test_paged_tiles_host.py looks at): some
of the heads against the plain 64-bit form, within bounds derived from the
arithmetic."""
import math

import pytest
import torch

import live_ref as R
import paged_ref as P
import paged_tiles as T
from test_gpu_paged import BF16, F16, F8, KIND_IDS, KINDS, make, running, words

pytestmark = pytest.mark.gpu
BEFORE, BEHIND = 2, 3                  # rows of nobody
DTYPES = pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
# keys or values; an infinite key's logit may be either infinity or NaN: not compared
BAD = pytest.mark.parametrize("side,bad", [(0, math.nan), (1, math.nan), (1, math.inf), (1, -math.inf)])


def some_of(H):
    """Heads to check: the first, the last and one between."""
    return sorted({0, H // 2 - 1, H - 1})


def query_heads(some, G):
    return [h * G + y for h in some for y in range(G)]


class Paged:
    def __init__(self, name, cache_type, dtype, D, seed=40):
        _, _, self.H, self.G, self.counts, self.lens, self.page, self.window, self.sinks = T.PAGED[name]
        self.cache, self.tables = make(cache_type, self.H, D, self.page, self.lens, seed=seed, spare=3)
        self.dtype, self.scale, self.st = dtype, T.SCALE[D], [BEFORE + x for x in running(self.counts)]
        self.rows = self.st[-1] + BEHIND
        self.q = torch.randn(self.rows, self.H * self.G, D, generator=torch.Generator().manual_seed(seed + 1)).to(dtype)
        self.some = some_of(self.H)

    def attend(self, **kw):
        return self.cache.attend(0, self.q.cuda(), words(self.tables), words(self.lens), starts=words(self.st),
                                 window=self.window, sinks=self.sinks, scale=self.scale, max_rows=max(self.counts), **kw)

    def check(self, room=lambda ref: ref):
        Hq = self.H * self.G
        lse = torch.full((Hq, self.rows), 77.0, device="cuda")
        out = torch.full((self.rows, Hq, self.cache.dim), 55.0, dtype=self.dtype, device="cuda")
        self.attend(lse=lse, out=out)
        buf, scales = self.cache.buf[:, :, :, self.some], self.cache.scales
        pages = P.values(buf, None if scales is None else scales[:, :, :, self.some])[0]
        kv = [P.gathered(pages, t, n) for t, n in zip(self.tables, self.lens)]
        spans, mine = P.rows_of(self.st, len(self.lens), self.rows), query_heads(self.some, self.G)
        ref = T.attend(self.q[:, mine].double(), kv, self.lens, spans, self.window, self.sinks, self.scale)
        P.check(out[:, mine], lse[mine], room(ref), spans, self.dtype, 55.0, 77.0)
        return out, lse

    def hide_pages(self, gone):
        """The table entries `gone` name nothing; page 0, which is read in their
        place, is no sequence's and holds NaN."""
        for s, e, word in gone:
            self.tables[s][e] = word
        free = [i for i in range(self.cache.pages) if not any(i in t for t in self.tables)]
        if 0 not in free:
            self.cache.buf[:, free[0]] = self.cache.buf[:, 0]
            if self.cache.scales is not None:
                self.cache.scales[:, free[0]] = self.cache.scales[:, 0]
            self.tables = [[free[0] if i == 0 else i for i in t] for t in self.tables]
        if self.cache.scales is None:
            self.cache.buf[:, 0] = math.nan
        else:
            self.cache.scales[:, 0] = 255


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name", T.PAGED)
def test_pages(ctx, name, cache_type, dtype, D):
    case = Paged(name, cache_type, dtype, D)
    out, _ = case.check()
    torch.full_like(out, 9.0)                     # what the next allocation may find
    new = case.attend()
    first, last = case.st[0], case.st[-1]
    assert R.same(new[first:last], out[first:last]) and not new[:first].any() and not new[last:].any()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name", ["256 long", "256 window", "256 mixed", "128 join", "128 long", "64 join"])
def test_missing_pages(ctx, name, cache_type, dtype, D):
    """Pages that are none in front of the rows, among them, at the start and the
    whole of a sequence, whatever page 0 holds."""
    case = Paged(name, cache_type, dtype, D, seed=42)
    n = len(case.tables[0])
    gone = [(0, 0, -1), (0, n // 3, 10 ** 6), (0, n // 2, -2 ** 31), (0, n - 2, 2 ** 31 - 1)]
    if len(case.tables) > 1:
        gone += [(len(case.tables) - 1, e, -1) for e in range(len(case.tables[-1]))]
    case.hide_pages(gone)
    out, _ = case.check()
    assert torch.isfinite(out).all()


@BAD
@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name,D", [("256 long", 128), ("256 window", 64), ("256 short", 64), ("128 join", 128), ("128 window", 64),
                                    ("64 join", 128)])
def test_pages_that_are_not_finite(ctx, name, D, cache_type, dtype, side, bad):
    """One slot's keys or values are not finite (of 8-bit pages a block of NaN), on
    the last head; rows that see it get what the formula gives, the others keep
    their values."""
    case = Paged(name, cache_type, dtype, D, seed=44)
    j = case.lens[0] - case.counts[0] // 2 - 1             # seen by about half of the rows
    page, head = case.tables[0][j // case.page], case.H - 1
    if cache_type == F8:
        case.cache.scales[0, page, side, head, j % case.page, 1] = 255
    else:
        case.cache.buf[0, page, side, head, j % case.page, 37] = bad
    out, _ = case.check()
    assert not torch.isfinite(out[:, head * case.G:]).all() and torch.isfinite(out[:, :head * case.G]).all()


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name,D", [("256 long", 64), ("256 mixed", 128), ("128 join", 64), ("128 long", 128), ("64 join", 128)])
def test_pages_of_large_logits_and_values(ctx, name, D, cache_type, dtype):
    """Logits in the hundreds, and values whose sums pass the end of the type."""
    case = Paged(name, cache_type, dtype, D, seed=46)
    case.scale = 4.0
    case.check()
    cache, big = case.cache, {BF16: 2.0 ** 126, F16: 2.0 ** 14, F8: 2.0 ** 14 if dtype == F16 else 2.0 ** 118}[cache_type]
    if cache_type == F8:
        cache.buf.random_(0, 256)
        cache.buf[(cache.buf & 127) == 127] = 0x7e
        cache.scales[:, :, 0].fill_(110)
        cache.scales[:, :, 1].fill_(127 + int(math.log2(big)) - 8)
    else:
        cache.buf[:, :, 1] = torch.rand(cache.buf[:, :, 1].shape, device="cuda").to(dtype) * big
    room = (lambda ref: ref) if cache_type == F16 else lambda ref: T.small_weights(ref, dtype)
    case.check(room)
    case.scale = T.SCALE[D] / 64                  # many slots of about the same weight
    case.check(room)


class Prompts:
    def __init__(self, name, dtype, D, seed=50):
        _, _, self.H, self.G, self.counts, self.window, self.sinks = T.PROMPTS[name]
        H, G = self.H, self.G
        self.dtype, self.scale, self.st = dtype, T.SCALE[D], [BEFORE + x for x in running(self.counts)]
        self.rows = self.st[-1] + BEHIND
        self.x = torch.randn(self.rows, H * (G + 2), D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
        self.q, self.k, self.v = self.x[:, :H * G], self.x[:, H * G:H * G + H], self.x[:, H * G + H:]
        self.some = some_of(H)

    def attend(self, **kw):
        from provekv_amd.paged import attend_prompts
        return attend_prompts(self.q, self.k, self.v, words(self.st), window=self.window, sinks=self.sinks, scale=self.scale,
                              max_rows=max(self.counts), **kw)

    def check(self, room=lambda ref: ref):
        Hq = self.H * self.G
        lse = torch.full((Hq, self.rows), 77.0, device="cuda")
        out = torch.full((self.rows, Hq, self.q.shape[2]), 55.0, dtype=self.dtype, device="cuda")
        self.attend(lse=lse, out=out)
        spans, mine = P.rows_of(self.st, len(self.counts), self.rows), query_heads(self.some, self.G)
        k, v = (t[:, self.some].cpu().double().transpose(0, 1) for t in (self.k, self.v))
        kv = [(k[:, a:a + m], v[:, a:a + m], torch.ones(m, dtype=torch.bool)) for a, m in spans]
        ref = T.attend(self.q[:, mine].cpu().double(), kv, self.counts, spans, self.window, self.sinks, self.scale)
        P.check(out[:, mine], lse[mine], room(ref), spans, self.dtype, 55.0, 77.0)
        return out, lse


@pytest.mark.parametrize("D", [64, 128])
@DTYPES
@pytest.mark.parametrize("name", T.PROMPTS)
def test_prompts(ctx, name, dtype, D):
    case = Prompts(name, dtype, D)
    out, _ = case.check()
    torch.full_like(out, 9.0)
    new = case.attend()
    first, last = case.st[0], case.st[-1]
    assert R.same(new[first:last], out[first:last]) and not new[:first].any() and not new[last:].any()


@BAD
@DTYPES
@pytest.mark.parametrize("name,D", [("256", 64), ("256 long", 128), ("256 window", 128), ("128", 128), ("128 long", 64), ("64 long", 128)])
def test_prompts_that_are_not_finite(ctx, name, D, dtype, side, bad):
    case = Prompts(name, dtype, D, seed=52)
    row = case.st[0] + case.counts[0] * 2 // 3
    (case.v if side else case.k)[row, case.H - 1, 9] = bad
    out, _ = case.check()
    head = (case.H - 1) * case.G
    assert torch.isfinite(out[:row]).all() and torch.isfinite(out[:, :head]).all() and not torch.isfinite(out[row, head:]).all()


@DTYPES
@pytest.mark.parametrize("name,D", [("256 long", 64), ("256", 128), ("128", 64), ("128 long", 128), ("64 long", 128)])
def test_prompts_of_large_logits_and_values(ctx, name, D, dtype):
    case = Prompts(name, dtype, D, seed=54)
    case.scale = 4.0
    case.check()
    case.v.uniform_(0.0, {BF16: 2.0 ** 126, F16: 2.0 ** 14}[dtype])
    room = (lambda ref: ref) if dtype == F16 else lambda ref: T.small_weights(ref, dtype)
    case.check(room)
    case.scale = T.SCALE[D] / 64
    case.check(room)


@DTYPES
@pytest.mark.parametrize("name", ["256 long", "256 window", "128", "64 long"])
def test_captured(ctx, name, dtype):
    """A captured call replayed with other starts and rows, eager calls between."""
    case = Prompts(name, dtype, 128, seed=56)
    from provekv_amd.paged import attend_prompts
    st, out = words(case.st), torch.zeros(case.rows, case.H * case.G, 128, dtype=dtype, device="cuda")

    def call(out):
        return attend_prompts(case.q, case.k, case.v, st, window=case.window, sinks=case.sinks, max_rows=max(case.counts),
                              out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out)
    for i in range(4):
        st.copy_(words([min(x + 5 * i, case.rows) if x == case.st[0] else max(x - 7 * i, case.st[0] + 5 * i) for x in case.st]))
        case.x.normal_()
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert R.same(out, call(torch.full_like(out, 3.0)))


@pytest.mark.parametrize("cache_type,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("name", ["256 long", "256 mixed", "128 join", "64 join"])
def test_repeated(ctx, name, cache_type, dtype):
    """The same call gives the same bits."""
    case = Paged(name, cache_type, dtype, 128, seed=58)
    first = case.attend()
    for _ in range(3):
        assert R.same(case.attend(), first)

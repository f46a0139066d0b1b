"""Attention over live caches (f32, bf16, f16 and 4-bit): every output against a
plain 64-bit form within bounds derived from the arithmetic (live_ref.py)."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KINDS = [("plain", F32), ("plain", BF16), ("plain", F16), ("fp4", F32), ("fp4", BF16), ("fp4", F16)]
KIND_IDS = ["f32", "bf16", "f16", "fp4-f32", "fp4-bf16", "fp4-f16"]


def make(kind, dtype, C, H, T, D, seed=0, layers=1):
    """(cache, keys, values as f64 of layer `layers` - 1 on the CPU)"""
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(C, layers, 2, H, T, D, generator=g)
    x[:, :, 0] *= torch.exp(0.4 * torch.randn(H, 1, D, generator=g))
    if kind == "plain":
        cache = DeviceKVCache.over(x.to(dtype).cuda())
        full = cache.buf.cpu().double()
    else:
        cache = FourBitKVCache(layers, H, T, D, copies=C)
        cache.store(x[:, :, 0].cuda(), x[:, :, 1].cuda(), 0)
        full = R.fp4_values(cache.codes, cache.scales)
    return cache, full[:, -1, 0], full[:, -1, 1]


def run(cache, dtype, k, v, lens, n, G, layer=0, q_lens=None, window=0, sinks=0, scale=None, seed=1, check_weights=True,
        max_len=None):
    """One call with every output, checked."""
    C, H, T, D = k.shape
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(C, n, H * G, D, generator=g).to(dtype)
    before = torch.rand(C, H, T, generator=g)
    w, lse = before.cuda(), torch.full((C, H * G, n), 77.0, device="cuda")
    out = torch.full((C, n, H * G, D), 55.0, dtype=dtype, device="cuda")
    d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    d_ql = None if q_lens is None else torch.tensor(q_lens, dtype=torch.int32, device="cuda")
    got = cache.attend(layer, q.cuda(), d_lens, q_lens=d_ql, window=window, sinks=sinks, scale=scale,
                       weights=w if check_weights else None, lse=lse, out=out, max_len=max_len)
    assert got is out
    ql = [n] * C if q_lens is None else q_lens
    ref = R.attend(q.double(), k, v, lens, ql, window, sinks, 1 / math.sqrt(D) if scale is None else scale)
    o = out.cpu().double()
    bound = R.out_bound(ref, dtype)
    for c in range(C):
        assert R.same(o[c, ql[c]:], torch.full_like(o[c, ql[c]:], 55.0)), "padding rows were written"
        assert R.same(lse[c, :, ql[c]:].cpu(), torch.full_like(lse[c, :, ql[c]:].cpu(), 77.0))
        err = (o[c, :ql[c]] - ref["out"][c, :ql[c]]).abs() - bound[c, :ql[c]]
        assert not (err > 0).any() and not torch.isnan(err).any(), f"copy {c}: out over its bound by {err.max()}"
        a, b = lse[c, :, :ql[c]].cpu().double(), ref["lse"][c, :, :ql[c]]
        assert R.same(torch.isinf(a), torch.isinf(b))
        fin = torch.isfinite(b)
        assert ((a - b).abs()[fin] <= R.lse_bound(ref)[c, :, :ql[c]][fin]).all()
    if check_weights:
        err = (w.cpu().double() - before.double() - ref["weights"]).abs() - R.weights_bound(ref, before, n * G)
        assert not (err > 0).any() and not torch.isnan(err).any(), f"weights over their bound by {err.max()}"
        # slots that no row sees keep their bits
        assert R.same(w.cpu()[ref["weights"] == 0], before[ref["weights"] == 0])
    return out


SIZES = [  # rows, group, capacity, lengths
    (1, 1, 1, [1]), (1, 1, 40, [0, 1, 40]), (1, 4, 70, [63, 64, 65]), (1, 3, 300, [257, 300]), (1, 16, 130, [130]),
    (1, 17, 100, [99]), (2, 8, 129, [129, 1]), (5, 3, 200, [130, 4, 0]), (16, 1, 64, [64, 16]), (33, 1, 90, [90, 20]),
    (64, 2, 150, [150, 100]), (130, 1, 257, [257, 131]), (200, 3, 333, [333, 150]),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n,G,T,lens", SIZES)
def test_sizes(ctx, n, G, T, lens, kind, dtype, D):
    cache, k, v = make(kind, dtype, len(lens), 2, T, D, seed=n + T)
    run(cache, dtype, k, v, lens, n, G)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 3), (64, 0), (65, 4), (100, 64), (1000, 5), (3, 500)])
@pytest.mark.parametrize("n,G", [(1, 4), (6, 2), (90, 1)])
def test_windows(ctx, n, G, window, sinks, kind, dtype):
    lens = [400, 211, 30]
    cache, k, v = make(kind, dtype, 3, 2, 400, 64, seed=3)
    run(cache, dtype, k, v, lens, n, G, window=window, sinks=sinks)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n,G,D", [(3, 2, 64), (41, 3, 128), (150, 1, 64)])
def test_padded_rows(ctx, n, G, D, kind, dtype):
    """Ragged row counts: none, one, some, all; also more rows than slots."""
    cache, k, v = make(kind, dtype, 5, 2, 200, D, seed=4)
    run(cache, dtype, k, v, [200, 120, 77, 150, n // 2], n, G, q_lens=[0, 1, n // 2, n, n], window=50, sinks=2)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
def test_layer_scale_max_len(ctx, kind, dtype):
    cache, k, v = make(kind, dtype, 2, 3, 500, 128, seed=5, layers=3)
    run(cache, dtype, k, v, [310, 37], 1, 2, layer=2, scale=0.31, max_len=320)
    run(cache, dtype, k, v, [310, 37], 40, 2, layer=2, scale=0.02, max_len=310)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n,G", [(1, 4), (1, 1)])
def test_long(ctx, n, G, kind, dtype):
    """Enough slots that a row's are split over many workgroups."""
    cache, k, v = make(kind, dtype, 2, 1, 9001, 128, seed=6)
    run(cache, dtype, k, v, [9001, 4100], n, G)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
def test_few_rows_long(ctx, kind, dtype):
    cache, k, v = make(kind, dtype, 1, 1, 5000, 64, seed=7)
    run(cache, dtype, k, v, [5000], 24, 2)
    run(cache, dtype, k, v, [5000], 3, 16, scale=0.5)
    run(cache, dtype, k, v, [4999], 9, 1, window=3000, sinks=4)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,G", [(1, 2), (4, 2), (70, 1)])
def test_hidden_slots_may_hold_anything(ctx, n, G, dtype, bad):
    """Slots behind the length, behind a row's own slot and outside its window
    hold infinities and NaN: rows that do not see them do not change."""
    cache, k, v = make("plain", dtype, 2, 2, 300, 64, seed=8)
    lens, window, sinks = [260, 150], 40, 3
    for c in range(2):
        first = lens[c] - n
        hidden = torch.ones(300, dtype=torch.bool)
        for i in range(n):
            hidden &= ~R.seen(first + i, 300, window, sinks)
        cache.buf[c, 0, :, :, hidden.cuda()] = bad
    run(cache, dtype, k, v, lens, n, G, window=window, sinks=sinks)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("side", [0, 1])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [4, 70, 140])
def test_bad_slot_reaches_only_rows_that_see_it(ctx, n, dtype, side, bad):
    """One bad row inside a tile that some query rows see and others do not."""
    T, window, sinks = 300, 40, 2
    lens = [280]
    cache, k, v = make("plain", dtype, 1, 2, T, 64, seed=9)
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, n, 2, 64, generator=g).to(dtype).cuda()
    clean = cache.attend(0, q, 280, window=window, sinks=sinks)
    slot = 280 - n // 2
    cache.buf[0, 0, side, :, slot] = bad
    w = torch.zeros(1, 2, T, device="cuda")
    got = cache.attend(0, q, 280, window=window, sinks=sinks, weights=w)
    for i in range(n):
        if bool(R.seen(lens[0] - n + i, T, window, sinks)[slot]):
            assert not torch.isfinite(got[0, i]).any() if side == 1 else torch.isnan(got[0, i]).any()
        else:
            assert R.same(got[0, i], clean[0, i])
    far = R.seen(280 - n, T, window, sinks) & ~R.seen(slot, T, window, sinks)
    if side == 0 and far.any():
        assert torch.isfinite(w.cpu()[0, 0][far & (torch.arange(T) < slot - window)]).all()


@pytest.mark.parametrize("n", [3, 70])
def test_fp4_nan_block_reaches_only_rows_that_see_it(ctx, n):
    T, window = 200, 30
    cache, k, v = make("fp4", BF16, 1, 1, T, 64, seed=10)
    q = torch.randn(1, n, 2, 64, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    clean = cache.attend(0, q, T, window=window)
    slot = T - n // 2 - 1
    cache.scales[0, 0, 1, 0, slot, 1] = 255
    got = cache.attend(0, q, T, window=window)
    for i in range(n):
        if bool(R.seen(T - n + i, T, window, 0)[slot]):
            assert torch.isnan(got[0, i, :, 32:]).all() and R.same(got[0, i, :, :32], clean[0, i, :, :32])
        else:
            assert R.same(got[0, i], clean[0, i])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 50])
def test_every_logit_minus_infinity(ctx, n, dtype):
    """A row whose visible logits are all -inf is an empty row: 0, -inf, no
    weight (4-bit keys are finite or NaN)."""
    from provekv_amd.pool import DeviceKVCache
    buf = torch.randn(1, 1, 2, 1, 80, 64, generator=torch.Generator().manual_seed(3))
    buf[0, 0, 0, 0, :, 5] = -math.inf
    cache = DeviceKVCache.over(buf.to(dtype).cuda())
    q = torch.zeros(1, n, 1, 64)
    q[..., 5] = 1.0
    w, lse = torch.ones(1, 1, 80, device="cuda"), torch.zeros(1, 1, n, device="cuda")
    # other channels: 0 * finite = 0, so each logit is exactly -inf
    out = cache.attend(0, q.to(dtype).cuda(), 80, weights=w, lse=lse)
    assert R.same(out, torch.zeros_like(out)) and (lse == -math.inf).all() and (w == 1).all()


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n", [1, 60])
def test_large_logits(ctx, n, kind, dtype):
    """Logits to some hundreds: one slot takes nearly everything."""
    cache, k, v = make(kind, dtype, 1, 2, 300, 64, seed=11)
    run(cache, dtype, k, v, [300], n, 2, scale=8.0)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n", [1, 40])
def test_strides(ctx, n, kind, dtype):
    """q cut out of a fused projection, out a view of [copies, heads, rows, dim],
    weights with gaps; a q of odd alignment is copied by the call."""
    C, H, G, D, T = 2, 2, 3, 64, 120
    cache, k, v = make(kind, dtype, C, H, T, D, seed=12)
    lens = torch.tensor([120, 50], dtype=torch.int32, device="cuda")
    fused = torch.randn(C, n, H * G + 4, D, device="cuda").to(dtype)
    q = fused[:, :, 2:2 + H * G]
    want = cache.attend(0, q.contiguous(), lens)
    out = torch.zeros(C, H * G, n, D, dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    wide = torch.zeros(C, H + 1, T + 9, device="cuda")
    got = cache.attend(0, q, lens, out=out, weights=wide[:, :H, :T])
    assert got is out and R.same(out, want)
    w = torch.zeros(C, H, T, device="cuda")
    cache.attend(0, q, lens, weights=w)
    assert R.same(wide[:, :H, :T], w) and not wide[:, H:].any() and not wide[:, :, T:].any()
    odd = torch.randn(C * n * H * G * D + 1, device="cuda").to(dtype)[1:].view(C, n, H * G, D)
    odd.copy_(q)
    assert R.same(cache.attend(0, odd, lens), want)


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n,T", [(1, 6000), (1, 60), (70, 700)])
def test_same_bits_every_time(ctx, n, T, kind, dtype):
    cache, k, v = make(kind, dtype, 2, 2, T, 64, seed=13)
    q = torch.randn(2, n, 4, 64, device="cuda").to(dtype)
    runs = []
    for _ in range(3):
        w = torch.zeros(2, 2, T, device="cuda")
        runs.append((cache.attend(0, q, T, weights=w), w))
    for o, w in runs[1:]:
        assert R.same(o, runs[0][0]) and R.same(w, runs[0][1])


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("n", [1, 40])
def test_captured_with_new_lengths(ctx, n, kind, dtype):
    """A captured call replays with other lengths and queries; eager calls between."""
    cache, k, v = make(kind, dtype, 2, 2, 2000, 64, seed=14)
    q = torch.randn(2, n, 4, 64, device="cuda").to(dtype)
    lens = torch.tensor([2000, 1500], dtype=torch.int32, device="cuda")
    w = torch.zeros(2, 2, 2000, device="cuda")
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.attend(0, q, lens, weights=w, out=out)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.attend(0, q, lens, weights=w, out=out)
    for a, b in ((2000, 1500), (1, 77), (n, 1999), (640, 0)):
        lens.copy_(torch.tensor([a, b], dtype=torch.int32))
        q.copy_(torch.randn(q.shape).to(dtype))
        w.zero_()
        g.replay()
        torch.cuda.synchronize()
        got_o, got_w = out.clone(), w.clone()
        w2 = torch.zeros_like(w)
        want = cache.attend(0, q, lens, weights=w2)
        assert R.same(got_o, want) and R.same(got_w, w2)


def test_side_stream_and_two_calls_at_once(ctx):
    cache, k, v = make("plain", BF16, 2, 4, 3000, 128, seed=15)
    q = [torch.randn(2, 1, 8, 128, device="cuda").to(BF16) for _ in range(4)]
    want = [cache.attend(0, x, 3000) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [cache.attend(0, x, 3000, stream=streams[i % 2]) for i, x in enumerate(q)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert R.same(a, b)


def test_shared_pool_view(ctx):
    """Copies that share one memory (copy stride 0) through the C entry."""
    import ctypes as C
    from provekv_amd import _lib as L
    cache, k, v = make("plain", BF16, 1, 2, 90, 64, seed=16)
    q = torch.randn(3, 1, 4, 64, device="cuda").to(BF16)
    out = torch.empty_like(q)
    lens = torch.tensor([90, 5, 33], dtype=torch.int32, device="cuda")
    view = cache._view(0)
    view.copies, view.copy_stride = 3, 0
    op = L.AttendOp(view, q.data_ptr(), out.data_ptr(), 256, 256, 64, 256, 256, 64, lens.data_ptr(), None, None, None, 0,
                    0, None, 0, 0.125, L.DT_BF16, 4, 1, 0, 0, 0, 0)
    need = L.lib().pkv_attend_workspace(C.byref(op))
    work = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    op.d_workspace, op.workspace_bytes = work.data_ptr(), need
    assert L.lib().pkv_attend(ctx.ptr, C.byref(op), torch.cuda.current_stream().cuda_stream) == 0
    for c, n in enumerate((90, 5, 33)):
        assert R.same(out[c:c + 1], cache.attend(0, q[c:c + 1], n))


def test_out_of_range_lengths_are_taken_into_range(ctx):
    cache, k, v = make("plain", BF16, 2, 2, 100, 64, seed=17)
    q = torch.randn(2, 3, 2, 64, device="cuda").to(BF16)
    big = cache.attend(0, q, torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda"),
                       q_lens=torch.tensor([99, 3], dtype=torch.int32, device="cuda"))
    want = cache.attend(0, q, torch.tensor([100, 0], dtype=torch.int32, device="cuda"))
    assert R.same(big, want) and not want[1].any()


def test_offsets_past_32_bits(ctx):
    """A cache of more than 2^32 bytes and elements; the copy read lies behind them."""
    from provekv_amd.pool import DeviceKVCache
    C, H, T, D = 3, 8, 1 << 20, 128
    cache = DeviceKVCache(1, H, T, D, dtype=BF16, copies=C)
    cache.buf[2, 0, :, 7, T - 700:].normal_()
    x = cache.buf[2, 0, :, 7, T - 700:].cpu().double()
    q = torch.zeros(C, 2, H, D)
    q[2, :, 7] = torch.randn(2, D)
    q = q.to(BF16)
    out = cache.attend(0, q.cuda(), torch.tensor([0, 0, T], dtype=torch.int32, device="cuda"), window=600)
    ref = R.attend(q[2:, :, 7:].double(), x[:1].unsqueeze(1), x[1:].unsqueeze(1), [700], [2], 600, 0, 1 / math.sqrt(D))
    err = (out[2:, :, 7:].cpu().double() - ref["out"]).abs()
    assert (err <= R.out_bound(ref, BF16)).all() and not out[:2].any()


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,heads,T,window", [(1, 128, 1, 300, 0), (3, 40, 1, 130, 64), (700, 1, 1, 1500, 256),
                                               (300, 4, 5, 700, 0), (90, 2, 12, 1300, 0)])
def test_wide_groups_and_many_rows(ctx, n, G, heads, T, window, kind, dtype, D):
    """Row tiles of both kinds, shares of slots and of rows, weights on top."""
    cache, k, v = make(kind, dtype, 2, heads, T, D, seed=20)
    w = torch.zeros(2, heads, T, device="cuda")
    lens, ql = [T, T - T // 3], [n, n - n // 4]
    q = torch.randn(2, n, heads * G, D, generator=torch.Generator().manual_seed(2)).to(dtype)
    lens_d, ql_d = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lens, ql))
    out = cache.attend(0, q.cuda(), lens_d, q_lens=ql_d, window=window, sinks=3, weights=w)
    some = [0, 1, n // 2, n - n // 4 - 1]           # the plain form of a few rows; all rows' weights add up to their number
    for c in range(2):
        for i in sorted({i for i in some if i < ql[c]}):
            ref = R.attend(q[c:c + 1, i:i + 1].double(), k[c:c + 1], v[c:c + 1], [lens[c] - ql[c] + i + 1], [1], window, 3,
                           1 / math.sqrt(D))
            err = (out[c:c + 1, i:i + 1].cpu().double() - ref["out"]).abs() - R.out_bound(ref, dtype)
            assert not (err > 0).any() and not torch.isnan(err).any(), (c, i, float(err.max()))
        total = w[c].sum(-1).cpu().double()
        assert ((total - ql[c] * G).abs() <= ql[c] * G * 2.0 ** -14).all()
        assert not out[c, ql[c]:].any()


@pytest.mark.parametrize("kind,dtype", KINDS, ids=KIND_IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 21])
def test_odd_heads_and_slots(ctx, n, kind, dtype, D):
    """Odd heads x slots: the values' scale bytes start at any row's boundary."""
    cache, k, v = make(kind, dtype, 3, 3, 47, D, seed=22, layers=3)
    run(cache, dtype, k, v, [47, 13, 46], n, 2, layer=2, window=9, sinks=1)


@pytest.mark.parametrize("n", [1, 40])
def test_many_heads(ctx, n):
    """Thousands of copies x heads."""
    cache, k, v = make("plain", BF16, 300, 16, 33, 64, seed=21)
    q = torch.randn(300, n, 16, 64, generator=torch.Generator().manual_seed(3)).to(BF16)
    out = cache.attend(0, q.cuda(), 33)
    for c, h in ((0, 0), (150, 7), (299, 15)):
        ref = R.attend(q[c:c + 1, :, h:h + 1].double(), k[c:c + 1, h:h + 1], v[c:c + 1, h:h + 1], [33], [n], 0, 0, 0.125)
        assert ((out[c:c + 1, :, h:h + 1].cpu().double() - ref["out"]).abs() <= R.out_bound(ref, BF16)).all()


@pytest.mark.parametrize("dtype", [F32, F16], ids=["f32", "f16"])
@pytest.mark.parametrize("n", [1, 40])
def test_infinite_query_over_4_bits(ctx, n, dtype):
    """A query of several terms with an infinity: logits are +inf or -inf as the
    keys' signs have it -- all +inf gives NaN, all -inf an empty row."""
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(1, 1, 70, 64)
    x = torch.ones(1, 1, 1, 70, 64)
    cache.store(x.cuda(), x.cuda(), 0)
    q = torch.zeros(1, n, 2, 64)
    q[:, :, 0, 3], q[:, :, 1, 3] = math.inf, -math.inf
    out = cache.attend(0, q.to(dtype).cuda(), 70)
    assert torch.isnan(out[:, :, 0]).all() and not out[:, :, 1].any()


def test_uninitialised_memory_behind_the_length(ctx):
    """A cache allocated and not cleared, filled slot by slot: NaN patterns
    behind the length never matter, for any row count."""
    from provekv_amd.pool import DeviceKVCache
    T, D = 300, 64
    for dtype in (BF16, F16, F32):
        cache = DeviceKVCache.over(torch.full((1, 1, 2, 2, T, D), math.nan, dtype=dtype, device="cuda"))
        x = torch.randn(2, 2, T, D, generator=torch.Generator().manual_seed(4)).to(dtype)
        for length in (1, 31, 64, 65, 255):
            cache.buf[0, 0, :, :, :length] = x[:, :, :length].cuda()
            for n in (1, 5, 20, 64, length):
                if n > length:
                    continue
                run(cache, dtype, x[0:1].double(), x[1:2].double(), [length], n, 2, seed=length + n)


def test_other_device_and_stream_refused(ctx):
    cache, _, _ = make("plain", BF16, 1, 1, 8, 64)
    q = torch.zeros(1, 1, 1, 64, dtype=BF16)
    with pytest.raises(ValueError):
        cache.attend(0, q, 8)
    with pytest.raises(ValueError):
        cache.attend(0, q.cuda(), torch.tensor([8], dtype=torch.int32))
    with pytest.raises(ValueError):
        cache.attend(0, q.cuda(), torch.tensor([8], device="cuda"))            # int64
    with pytest.raises(ValueError):
        cache.attend(0, q.cuda(), 8, out=q.cuda()[..., :32])
    with pytest.raises(ValueError):
        cache.attend(0, q.cuda(), 8, max_len=9)
    with pytest.raises(ValueError):
        cache.attend(0, q.cuda(), 8, weights=torch.zeros(1, 1, 9, device="cuda"))
    with pytest.raises(IndexError):
        cache.attend(1, q.cuda(), 8)
    from provekv_amd._lib import PkvError
    x = q.cuda()
    with pytest.raises(PkvError):
        cache.attend(0, x, 8, out=x)
    with pytest.raises(PkvError):
        cache.attend(0, x, 8, scale=0.0)

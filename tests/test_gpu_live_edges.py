"""Attention over live caches at the edges of sizes and values, against plain
64-bit forms."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def held(kind, dtype, x, copies):
    """(cache of `copies` times the rows x [1, 1, 2, heads, slots, dim], keys and
    values as it holds them in f64)"""
    from provekv_amd.pool import DeviceKVCache, FourBitKVCache
    if kind == "plain":
        cache = DeviceKVCache.over(x.to(dtype).cuda().repeat(copies, 1, 1, 1, 1, 1))
        full = x.to(dtype).double()
    else:
        cache = FourBitKVCache(1, *x.shape[3:], copies=copies)
        x = x.cuda().expand(copies, -1, -1, -1, -1, -1)
        cache.store(x[:, :, 0], x[:, :, 1], 0)
        full = R.fp4_values(cache.codes[:1], cache.scales[:1])
    return cache, full[:, 0, 0], full[:, 0, 1]


@pytest.mark.parametrize("copies,G,n", [(64, 32, 8192), (2, 128, 65537)])
def test_millions_of_rows(ctx, copies, G, n):
    """copies x query heads x rows of 2^24 and past it, with weights: prompts of
    many agents and heads."""
    from provekv_amd.pool import DeviceKVCache
    T, D, window = n, 64, 40
    assert copies * G * n >= 1 << 24
    x = torch.randn(1, 1, 2, 1, T, D, generator=torch.Generator().manual_seed(1)).to(BF16)
    cache = DeviceKVCache.over(x.cuda().repeat(copies, 1, 1, 1, 1, 1))
    q = torch.randn(1, n, 1, D, generator=torch.Generator().manual_seed(2)).to(BF16)
    w = torch.zeros(copies, 1, T, device="cuda")
    lens = torch.full((copies,), T, dtype=torch.int32, device="cuda")
    out = cache.attend(0, q.cuda().expand(copies, -1, G, -1), lens, window=window, weights=w)
    x = x.double()
    for i in (0, 1, 127, 128, n // 2, n - 1):
        ref = R.attend(q[:, i:i + 1].double(), x[:, 0, 0], x[:, 0, 1], [i + 1], [1], window, 0, 0.125)
        for c, g in ((0, 0), (copies - 1, G - 1), (copies // 2, 1)):
            err = (out[c:c + 1, i:i + 1, g:g + 1].cpu().double() - ref["out"]).abs()
            assert (err <= R.out_bound(ref, BF16)).all(), (i, c, g)
    # every row gives its slots 1 in all
    total = w.double().sum((1, 2)).cpu()
    assert ((total - n * G).abs() <= n * G * 2.0 ** -14).all()
    assert R.same(w[0], w[-1])


@pytest.mark.parametrize("gap", [17.0, 17.5])
@pytest.mark.parametrize("n,G", [(1, 1), (3, 4), (40, 1), (150, 1)])
def test_f16_small_weights_of_many_slots(ctx, n, G, gap):
    """A first slot `gap` nats ahead of all others, whose value is small: the
    others' weights, 2^-24.5 and 2^-25.2 of its own, are what the output is.
    They are rounded at 2^11 times their size (pkv_attend.hip): half a step,
    2^-11 of them, or 2^-25 for those below 2^-14, here 2^-10 of them at most
    (2^-14.3 is the smallest).  No part of the bound grows with the slots."""
    from provekv_amd.pool import DeviceKVCache
    C, H, T, D = 96, 8, 4096, 64          # as many heads as fill the chip: a row is not split over many workgroups
    cache = DeviceKVCache(1, H, T, D, dtype=F16, copies=C)
    v = (32 + 32 * torch.rand(T, D, generator=torch.Generator().manual_seed(1))).to(F16)
    v[0] = 0
    cache.buf[:, 0, 0, :, 0, 5] = gap
    cache.buf[:, 0, 1] = v.cuda()
    q = torch.zeros(C, n, H * G, D, dtype=F16)
    q[..., 5] = 1.0
    out = cache.attend(0, q.cuda(), torch.full((C,), T, dtype=torch.int32, device="cuda"), scale=1.0).cpu().double()
    k = torch.zeros(1, 1, T, D, dtype=torch.float64)
    k[..., 0, 5] = gap
    ref = R.attend(q[:1, :, :1].double(), k, v.double().view(1, 1, T, D), [T], [n], 0, 0, 1.0)
    h, u = 2.0 ** -11, 2.0 ** -24
    rel = 2 * ref["dev"].unsqueeze(-1) * u + 4 * (T + 16) * u + 2 * h
    bound = h * ref["out"] + rel * ref["mass"]
    err = (out - ref["out"]).abs() - bound
    assert not (err > 0).any() and not torch.isnan(err).any(), float(((out - ref["out"]).abs() / ref["out"]).max())


@pytest.mark.parametrize("kind,dtype", [("plain", F32), ("plain", BF16), ("fp4", F32), ("fp4", BF16)],
                         ids=["f32", "bf16", "fp4-f32", "fp4-bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,G,copies", [(1, 1, 1), (1, 1, 400), (5, 3, 2), (40, 1, 2), (40, 1, 400), (300, 2, 1)])
def test_values_near_the_types_largest(ctx, n, G, copies, D, kind, dtype):
    """Means of values up to 2^126: sums over thousands of slots, before they are
    divided, stay finite."""
    T = 3000
    x = torch.randn(1, 1, 2, 1, T, D, generator=torch.Generator().manual_seed(2))
    x[:, :, 1] = (0.25 + 0.75 * torch.rand(x[:, :, 1].shape, generator=torch.Generator().manual_seed(3))) * 2.0 ** 126
    cache, k, v = held(kind, dtype, x, copies)
    q = torch.randn(1, n, G, D, generator=torch.Generator().manual_seed(4)).to(dtype)
    w = torch.zeros(copies, 1, T, device="cuda")
    lse = torch.zeros(copies, G, n, device="cuda")
    out = cache.attend(0, q.cuda().expand(copies, -1, -1, -1), T, weights=w, lse=lse)
    ref = R.attend(q.double(), k, v, [T], [n], 0, 0, 1 / math.sqrt(D))
    for c in {0, copies - 1}:
        err = (out[c:c + 1].cpu().double() - ref["out"]).abs()
        assert (err <= R.out_bound(ref, dtype)).all()
        assert ((lse[c:c + 1].cpu().double() - ref["lse"]).abs() <= R.lse_bound(ref)).all()
        err = (w[c:c + 1].cpu().double() - ref["weights"]).abs()
        assert (err <= R.weights_bound(ref, torch.zeros(1, 1, T), n * G)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("n,G,T", [(1, 1, 60), (1, 4, 3000), (4, 2, 300), (16, 1, 300), (17, 1, 300), (140, 2, 400)])
def test_infinite_values_keep_their_sign(ctx, n, G, T, window, D, dtype):
    """sum w_j v_j with infinities among the values that a row sees: inf with
    their sign, NaN where both signs meet or a NaN is among them, and the other
    channels and rows as with 0 in those places."""
    x = torch.randn(1, 1, 2, 2, T, D, generator=torch.Generator().manual_seed(5))
    bad = [(3, 1, math.inf), (3, 7, -math.inf), (T // 2, D - 1, -math.inf), (T - 1 - n // 2, 1, math.inf),
           (T - 1 - n // 2, 7, math.inf), (T - 1 - n // 3, 33, math.inf), (T - 1, 34, -math.inf), (T - 9, 40, math.nan)]
    for slot, d, _ in bad:
        x[0, 0, 1, :, slot, d] = 0
    cache, k, v = held("plain", dtype, x, 1)
    q = (0.2 * torch.randn(1, n, 2 * G, D, generator=torch.Generator().manual_seed(6))).to(dtype)
    ref = R.attend(q.double(), k, v, [T], [n], window, 2, 1 / math.sqrt(D))
    for slot, d, value in bad:
        cache.buf[0, 0, 1, 1, slot, d] = value        # the second head's
    lse = torch.zeros(1, 2 * G, n, device="cuda")
    got = cache.attend(0, q.cuda(), T, window=window, sinks=2, lse=lse).cpu().double()
    want = ref["out"].clone()
    for i in range(n):
        see = R.seen(T - n + i, T, window, 2)
        for slot, d, value in bad:
            if see[slot]:
                want[0, i, G:, d] += value
    assert R.same(torch.isnan(got), torch.isnan(want)) and R.same(got.isposinf(), want.isposinf())
    assert R.same(got.isneginf(), want.isneginf())
    fin = torch.isfinite(want)
    assert ((got - want).abs()[fin] <= R.out_bound(ref, dtype)[fin]).all()
    assert ((lse.cpu().double() - ref["lse"]).abs() <= R.lse_bound(ref)).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,T", [(1, 28), (3, 27), (40, 60), (200, 62)])
def test_same_bits_whatever_the_launch_is_sized_by(ctx, n, T, dtype):
    """Calls that are cut alike give the same bits for any max_len and capacity."""
    from provekv_amd.pool import DeviceKVCache
    x = torch.randn(1, 1, 2, 2, T, 64, generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    q = torch.randn(1, n, 4, 64, generator=torch.Generator().manual_seed(8)).to(dtype).cuda()
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    first = None
    for room, max_len in ((T, T), (T + 1, T), (2 * T, T), (2 * T, None)):
        buf = torch.zeros(1, 1, 2, 2, room, 64, dtype=dtype, device="cuda")
        buf[:, :, :, :, :T] = x
        cache = DeviceKVCache.over(buf)
        w, lse = torch.zeros(1, 2, room, device="cuda"), torch.zeros(1, 4, n, device="cuda")
        got = [cache.attend(0, q, lens, weights=w, lse=lse, max_len=max_len), lse, w[:, :, :T]]
        first = first or got
        for a, b in zip(got, first):
            assert R.same(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("n,G", [(1, 1), (7, 2), (40, 1), (300, 1)])
def test_infinite_and_large_values_together(ctx, n, G, dtype):
    T, D = 3000, 64
    x = torch.randn(1, 1, 2, 1, T, D, generator=torch.Generator().manual_seed(9))
    x[:, :, 1] = (0.25 + 0.75 * torch.rand(x[:, :, 1].shape, generator=torch.Generator().manual_seed(3))) * 2.0 ** 126
    x[0, 0, 1, 0, 11, 5] = x[0, 0, 1, 0, T - 1, 9] = 0
    cache, k, v = held("plain", dtype, x, 1)
    q = (0.2 * torch.randn(1, n, G, D, generator=torch.Generator().manual_seed(4))).to(dtype)
    ref = R.attend(q.double(), k, v, [T], [n], 0, 0, 1 / math.sqrt(D))
    cache.buf[0, 0, 1, 0, 11, 5], cache.buf[0, 0, 1, 0, T - 1, 9] = -math.inf, math.inf
    got = cache.attend(0, q.cuda(), T).cpu().double()
    want = ref["out"].clone()
    want[..., 5] = -math.inf
    want[0, n - 1, :, 9] = math.inf
    assert R.same(got.isposinf(), want.isposinf()) and R.same(got.isneginf(), want.isneginf())
    fin = torch.isfinite(want)
    assert ((got - want).abs()[fin] <= R.out_bound(ref, dtype)[fin]).all()


@pytest.mark.parametrize("n", [1, 20])
def test_int_lengths_are_the_launch_s_size(ctx, n):
    """A loop over int lengths gives what length tensors of that max_len give."""
    x = torch.randn(1, 1, 2, 2, 5000, 64, generator=torch.Generator().manual_seed(10))
    cache, _, _ = held("plain", BF16, x, 2)
    q = torch.randn(2, n, 4, 64, generator=torch.Generator().manual_seed(11)).to(BF16).cuda()
    for length in (0, 1, 100, 129, 1000, 4097, 5000, 6000):
        w, w2 = torch.zeros(2, 2, 2, 5000, device="cuda")
        got = cache.attend(0, q, length, weights=w)
        d = torch.full((2,), length, dtype=torch.int32, device="cuda")
        want = cache.attend(0, q, d, weights=w2, max_len=min(max(length, 1), 5000))
        assert R.same(got, want) and R.same(w, w2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 5, 40])
@pytest.mark.parametrize("power", [20, 24, 25, 26, 27])
def test_huge_logits(ctx, n, power, dtype):
    """A slot ahead by 2^20 .. 2^27 (in powers of two), where 32 bits hold an
    exponent to whole numbers and less: its value, and an lse within the logit's
    own rounding."""
    from provekv_amd.pool import DeviceKVCache
    C, H, T, D = 4, 16, 200, 64
    cache = DeviceKVCache(1, H, T, D, dtype=dtype, copies=C)
    g = torch.Generator().manual_seed(power)
    v = torch.randn(C, H, T, D, generator=g).to(dtype)
    cache.buf[:, 0, 1] = v.cuda()
    ahead = (2.0 ** (power - 13) * 0.69 * (0.5 + 0.5 * torch.rand(C, H, generator=g))).to(dtype)
    cache.buf[:, 0, 0, :, 7, 3] = ahead.cuda()
    q = torch.zeros(C, n, H, D, dtype=dtype)
    q[..., 3] = 8192.0
    lse = torch.zeros(C, H, n, device="cuda")
    w = torch.zeros(C, H, T, device="cuda")
    out = cache.attend(0, q.cuda(), T, scale=1.0, lse=lse, weights=w).cpu()
    # the only weight: 2^r with r what rounding the logit's exponent to 24 bits leaves (up to 2^-4 at 2^20), the sum as
    # well; of many rows it is rounded to the type, h at most, and the output once more: (1 + h)^2
    want, h = v[:, :, 7].unsqueeze(1).double(), R.HALF[dtype]
    rel = ((1 + h) ** 2 - 1 if n > 16 else h) + 2.0 ** -20
    assert ((out.double() - want).abs() <= want.abs() * rel).all()
    top = 8192.0 * ahead.double().unsqueeze(-1)
    assert ((lse.cpu().double() - top).abs() <= 4 * top * 2.0 ** -24).all()
    assert ((w.cpu().double()[:, :, 7] - n).abs() <= n * 2.0 ** -20).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("n", [1, 9, 40, 300])
def test_a_single_slot_gives_its_value(ctx, n, dtype):
    """A window of 1: every weight is 2^r / 2^r with r below 2^-18 (logits under
    2^6), which the types hold as 1; the value comes back as it was."""
    x = torch.randn(1, 1, 2, 3, 333, 64, generator=torch.Generator().manual_seed(12))
    cache, k, v = held("plain", dtype, x, 1)
    q = torch.randn(1, n, 6, 64, generator=torch.Generator().manual_seed(13)).to(dtype).cuda()
    w = torch.zeros(1, 3, 333, device="cuda")
    out = cache.attend(0, q, 333, window=1, weights=w).cpu().double()
    want = v[0, :, 333 - n:].permute(1, 0, 2).repeat_interleave(2, 1)
    err = (out[0] - want).abs()
    assert R.same(out[0], want) if dtype != F32 else (err <= want.abs() * 2.0 ** -17).all()
    assert ((w.cpu()[0, :, 333 - n:] - 2).abs() <= 2.0 ** -17).all() and not w[0, :, :333 - n].any()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("big", [False, True], ids=["", "large-values"])
@pytest.mark.parametrize("at", [0, 150])
@pytest.mark.parametrize("n,G", [(1, 1), (5, 2), (40, 1), (200, 1)])
def test_infinite_value_of_a_small_weight(ctx, n, G, at, big, dtype):
    """80 nats behind: a weight of 2^-115 still makes an infinity, and the rest
    is the slot ahead, also where the other values' sums pass the type's end
    (other weights: 2^-115 each, 300 of them below half a step)."""
    from provekv_amd.pool import DeviceKVCache
    if big and dtype == F16:
        return
    T, D = 300 + n, 64
    cache = DeviceKVCache(1, 2, T, D, dtype=dtype)
    cache.buf[:, 0, 0, :, at, 3] = 80.0
    cache.buf[:, 0, 1] = 2.0 ** 127 if big else 3.0
    cache.buf[:, 0, 1, :, 70, 9] = -math.inf
    q = torch.zeros(1, n, 2 * G, D, dtype=dtype)
    q[..., 3] = 1.0
    if big:      # more slots as far ahead, so that their values' sum is past the end
        cache.buf[:, 0, 0, :, at:at + 20, 3] = 80.0
    out = cache.attend(0, q.cuda(), T, scale=1.0).cpu().double()
    want = torch.full_like(out, 2.0 ** 127 if big else 3.0)
    want[..., 9] = -math.inf
    fin = torch.isfinite(want)
    assert R.same(out.isneginf(), want.isneginf())
    assert ((out - want).abs()[fin] <= want.abs()[fin] * (R.HALF[dtype] + 2.0 ** -18)).all()

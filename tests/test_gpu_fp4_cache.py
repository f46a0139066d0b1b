"""The 4-bit cache's store and load against the format's definition, bit for bit."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


def special(n, D, dtype, seed=0):
    """Rows of every magnitude, ties, zeros and subnormals."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, D, generator=g) * torch.pow(2.0, torch.randint(-20, 14, (n, 1), generator=g).float())
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 6.0, -0.25, -5.0, -0.75, 0.0, -0.0, 6.5, -7.0])
    x[0, :16], x[0, 16:32] = ties, ties * 0.999
    x[1] = 0.0
    if n > 2:
        x[2, :32] = ties.repeat(2) * 2.0 ** 10
        x[2, 32:64] = 1e-40 if dtype == torch.float32 else 0.0
    if n > 3 and dtype != torch.float16:
        x[3] = x[3].sign() * 2.0 ** -130
        x[3, :32] *= 2.0 ** 255
    if n > 4:
        x[4, :32] = float(torch.finfo(dtype).max)
        x[4, 32:64] = float(torch.finfo(dtype).tiny)
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 77])
def test_store_load(ctx, n, D, dtype):
    from provekv_amd.pool import FourBitKVCache
    C, L, H, T = 2, 3, 2, 100
    cache = FourBitKVCache(L, H, T, D, copies=C)
    x = special(2 * C * L * H * n, D, dtype).reshape(2, C, L, H, n, D)
    first = torch.tensor([100 - n, 3], dtype=torch.int32, device="cuda")
    cache.store(x[0].cuda(), x[1].cuda(), first)
    want = R.fp4_round(x)
    for out in (torch.float32, torch.bfloat16, torch.float16):
        keys, values = cache.load(first, n, dtype=out)
        for got, w in ((keys, want[0]), (values, want[1])):
            assert R.same(got.cpu(), w.to(out)), (dtype, out)
    # the codes themselves, in their places, and nothing else
    full = R.fp4_values(cache.codes, cache.scales)
    for c, f in ((0, 100 - n), (1, 3)):
        assert R.same(full[c, :, 0, :, f:f + n], want[0][c]) and R.same(full[c, :, 1, :, f:f + n], want[1][c])
        rest = torch.ones(T, dtype=torch.bool)
        rest[f:f + n] = False
        assert not cache.codes[c, :, :, :, rest.cuda()].any() and not cache.scales[c, :, :, :, rest.cuda()].any()


@pytest.mark.parametrize("D", [64, 128])
def test_odd_heads_and_slots(ctx, D):
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(3, 3, 11, D, copies=2)
    x = torch.randn(2, 2, 3, 3, 5, D, generator=torch.Generator().manual_seed(1))
    cache.store(x[0].cuda(), x[1].cuda(), 6)
    keys, values = cache.load(6, 5, dtype=torch.float32)
    want = R.fp4_round(x).float()
    assert R.same(keys, want[0]) and R.same(values, want[1])
    one, _ = cache.load(6, 5, layer=1, dtype=torch.float32)
    assert R.same(one, want[0][:, 1])


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_no_value_is_off_by_more_than_half_a_step(ctx, dtype):
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(1, 4, 500, 64)
    x = torch.randn(1, 1, 4, 500, 64, generator=torch.Generator().manual_seed(2)).to(dtype)
    cache.store(x.cuda(), None, 0)
    keys, values = cache.load(0, 500, dtype=torch.float32)
    step = torch.pow(2.0, cache.scales[:, :, 0].cpu().double() - 127).repeat_interleave(32, -1)
    assert ((keys.cpu().double() - x.double()).abs() <= step).all() and not values.any()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_nonfinite_block_becomes_nan(ctx, dtype, bad):
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(1, 1, 4, 128)
    x = torch.ones(1, 1, 1, 4, 128, dtype=dtype)
    x[..., 1, 37] = bad
    cache.store(x.cuda(), x.cuda(), 0)
    for t in cache.load(0, 4):
        t = t.cpu().float()
        assert torch.isnan(t[..., 1, 32:64]).all()
        t[..., 1, 32:64] = 1
        assert (t == 1).all()
    assert (cache.scales[0, 0, 0, 0, 1] == 255).tolist() == [False, True, False, False]


def test_rows_without_a_slot(ctx):
    """Counts, negative and late first slots: those rows are not stored, and load as 0."""
    from provekv_amd.pool import FourBitKVCache
    C, T, n = 5, 20, 6
    cache = FourBitKVCache(2, 3, T, 64, copies=C)
    x = torch.randn(C, 2, 3, n, 64, generator=torch.Generator().manual_seed(3))
    first = torch.tensor([-3, 17, 2 ** 31 - 1, 5, 6], dtype=torch.int32, device="cuda")
    counts = torch.tensor([6, 6, 6, 2, -1], dtype=torch.int32, device="cuda")
    cache.store(x.cuda(), x.cuda(), first, counts=counts)
    want = torch.zeros(C, 2, 3, T, 64, dtype=torch.float64)
    r = R.fp4_round(x)
    want[0, :, :, :3] = r[0, :, :, 3:]
    want[1, :, :, 17:] = r[1, :, :, :3]
    want[3, :, :, 5:7] = r[3, :, :, :2]
    full = R.fp4_values(cache.codes, cache.scales)
    assert R.same(full[:, :, 0], want) and R.same(full[:, :, 1], want)
    keys, _ = cache.load(first, n, counts=counts, dtype=torch.float32)
    assert not keys[2].any() and not keys[4].any() and not keys[3, :, :, 2:].any() and not keys[0, :, :, :3].any()
    assert R.same(keys[0, :, :, 3:].cpu().double(), r[0, :, :, 3:])


def test_one_layer_strided_rows_and_cache_target(ctx):
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(3, 4, 30, 64, copies=2)
    tok = torch.randn(2, 5, 3, 4, 64, device="cuda").to(torch.bfloat16)   # [copies, rows, q|k|v, heads, dim]
    k, v = (tok[:, :, i].permute(0, 2, 1, 3) for i in (1, 2))             # [copies, heads, rows, dim]
    cache.store(k, v, 7, layer=1)
    keys, values = cache.load(7, 5, layer=1)
    assert R.same(keys.cpu().double(), R.fp4_round(k)) and R.same(values.cpu().double(), R.fp4_round(v))
    assert not cache.codes[:, [0, 2]].any()
    vec = torch.randn(4 * 64).numpy()
    cache.append_key(2, 11, vec)
    cache.append_value(2, 12, vec)
    assert cache.seq_len() == 13 and cache.num_layers() == 3
    want = R.fp4_round(torch.from_numpy(vec).reshape(4, 64))
    full = R.fp4_values(cache.codes, cache.scales)
    assert R.same(full[1, 2, 0, :, 11], want) and R.same(full[0, 2, 1, :, 12], want)
    with pytest.raises(IndexError):
        cache.append_key(2, 30, vec)


def test_captured_append(ctx):
    from provekv_amd.pool import FourBitKVCache
    cache = FourBitKVCache(2, 2, 16, 64, copies=2)
    k, v = (torch.zeros(2, 2, 2, 1, 64, device="cuda") for _ in range(2))
    first = torch.zeros(2, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.store(k, v, first)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.store(k, v, first)
    want = torch.zeros(2, 2, 2, 2, 16, 64, dtype=torch.float64)
    for step in range(4):
        x = torch.randn(2, 2, 2, 2, 1, 64)
        k.copy_(x[0])
        v.copy_(x[1])
        first.copy_(torch.tensor([step, 15 - step], dtype=torch.int32))
        g.replay()
        r = R.fp4_round(x)
        for c, j in ((0, step), (1, 15 - step)):
            want[c, :, 0, :, j], want[c, :, 1, :, j] = r[0, c, :, :, 0], r[1, c, :, :, 0]
        torch.cuda.synchronize()
        if step == 0:
            cache.codes[:, :, :, :, 1:15] = 0
    assert R.same(R.fp4_values(cache.codes, cache.scales), want)

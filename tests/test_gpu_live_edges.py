"""Attention over live caches at the edges of sizes and values, against plain
64-bit forms."""
import math

import pytest
import torch

import live_ref as R

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("copies,G,n", [(64, 32, 8192), (2, 128, 65537)])
def test_millions_of_rows(ctx, copies, G, n):
    """copies x query heads x rows of 2^24 and past it, with weights: prompts of
    many agents and heads."""
    from provekv_amd.pool import DeviceKVCache
    T, D, window = n, 64, 40
    assert copies * G * n >= 1 << 24
    x = torch.randn(1, 1, 2, 1, T, D, generator=torch.Generator().manual_seed(1)).to(BF16).expand(copies, -1, -1, -1, -1, -1)
    cache = DeviceKVCache.over(x.contiguous().cuda())
    q = torch.randn(1, n, 1, D, generator=torch.Generator().manual_seed(2)).to(BF16)
    w = torch.zeros(copies, 1, T, device="cuda")
    out = cache.attend(0, q.cuda().expand(copies, -1, G, -1), torch.full((copies,), T, dtype=torch.int32, device="cuda"),
                       window=window, weights=w)
    x = x[:1].double()
    for i in (0, 1, 127, 128, n // 2, n - 1):
        ref = R.attend(q[:, i:i + 1].double(), x[:, 0, 0], x[:, 0, 1], [i + 1], [1], window, 0, 0.125)
        for c, g in ((0, 0), (copies - 1, G - 1), (copies // 2, 1)):
            err = (out[c:c + 1, i:i + 1, g:g + 1].cpu().double() - ref["out"]).abs()
            assert (err <= R.out_bound(ref, BF16)).all(), (i, c, g)
    # every row gives its slots 1 in all
    total = w.double().sum((1, 2)).cpu()
    assert ((total - n * G).abs() <= n * G * 2.0 ** -14).all()
    assert R.same(w[0], w[-1])

"""The call structs that live caches keep per shape, on caches in host memory: a
call there is refused, but only after its struct is made."""
import pytest
import torch

from provekv_amd.pool import DeviceKVCache, FourBitKVCache


def refused(call, *args, **kw):
    with pytest.raises(ValueError, match="not on a GPU"):
        call(*args, **kw)


@pytest.mark.parametrize("kind", ["plain", "fp4"])
def test_one_struct_for_a_loop_over_lengths(kind):
    """A decode loop that counts its tokens makes no struct per token."""
    if kind == "plain":
        cache = DeviceKVCache(2, 2, 600, 64, dtype=torch.bfloat16, device="cpu")
    else:
        cache = FourBitKVCache(2, 2, 600, 64, device="cpu")
    q = torch.zeros(1, 1, 4, 64, dtype=torch.bfloat16)
    w = torch.zeros(1, 2, 600)
    for n in range(1, 601):
        for layer in range(2):
            refused(cache.attend, layer, q, n)
            refused(cache.attend, layer, q, n, weights=w, window=100)
    assert len(cache._plans) == 4

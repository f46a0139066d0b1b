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


def test_lost_derivatives_are_refused():
    """Gradients and forward-mode tangents of queries and stored rows; not where
    nothing is recorded."""
    import torch.autograd.forward_ad as fwd
    cache = DeviceKVCache(1, 2, 10, 64, device="cpu")
    four = FourBitKVCache(1, 2, 10, 64, device="cpu")
    q, rows = torch.zeros(1, 3, 4, 64), torch.zeros(1, 2, 3, 64)
    leaf, leaf_rows = q.clone().requires_grad_(), rows.clone().requires_grad_()
    lost = [lambda x, r: cache.attend(0, x, 5), lambda x, r: four.attend(0, x, 5),
            lambda x, r: four.store(r, rows, 0, layer=0), lambda x, r: four.store(None, r, 0, layer=0)]
    for call in lost:
        with pytest.raises(ValueError, match="no backward pass"):
            call(leaf, leaf_rows)
        with torch.no_grad():
            refused(call, leaf, leaf_rows)
        refused(call, leaf.detach(), leaf_rows.detach())
        with fwd.dual_level():
            x, r = fwd.make_dual(q, torch.ones_like(q)), fwd.make_dual(rows, torch.ones_like(rows))
            with pytest.raises(ValueError, match="no forward-mode"):
                call(x, r)
            with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode"):
                call(x, r)
            refused(call, fwd.unpack_dual(x).primal, fwd.unpack_dual(r).primal)
            refused(call, q, rows)

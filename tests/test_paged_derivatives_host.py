"""Paged calls have no derivative: tensors that carry a gradient or a tangent are
refused, on the CPU, before anything is launched."""
import pytest
import torch
from torch.autograd import forward_ad

from provekv_amd.paged import PagedKVCache, attend_prompts

BF16 = torch.bfloat16


def calls(buf=None, **given):
    """Each call that reads or writes `buf`, or is given a tensor to write."""
    cache = PagedKVCache.over(torch.zeros(1, 4, 2, 2, 16, 64, dtype=BF16) if buf is None else buf)
    tables, lens = torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    q, rows = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(1, 3, 2, 64)
    yield lambda: cache.attend(0, q, tables, lens, **given)
    if given:
        yield lambda: attend_prompts(q, q[:, :2], q[:, :2], torch.zeros(2, dtype=torch.int32), **given)
    else:
        yield lambda: cache.store(rows, rows, tables, lens)
        yield lambda: cache.load(3, tables, lens)


def written():
    return [("out", torch.zeros(3, 4, 64, dtype=BF16)), ("lse", torch.zeros(4, 3))]


def test_pages_that_carry_a_gradient():
    buf = torch.zeros(1, 4, 2, 2, 16, 64, dtype=BF16, requires_grad=True)
    for call in calls(buf):
        with pytest.raises(ValueError, match="no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="not on a GPU"):
            call()
    for call in calls():
        with pytest.raises(ValueError, match="not on a GPU"):
            call()


@pytest.mark.parametrize("name,t", written(), ids=["out", "lse"])
def test_outputs_that_carry_a_gradient(name, t):
    for call in calls(**{name: t.clone().requires_grad_()}):
        with pytest.raises(ValueError, match="no backward pass"):
            call()
    for call in calls(**{name: t}):
        with pytest.raises(ValueError, match="not on a GPU"):
            call()


def test_tangents():
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in calls(dual(torch.zeros(1, 4, 2, 2, 16, 64, dtype=BF16))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        for name, t in written():
            for call in calls(**{name: dual(t)}):
                with pytest.raises(ValueError, match="forward-mode"):
                    call()

"""Eviction: caches longer than the selection holds in registers (32,768 slots),
and the filled length that a cache remembers."""
import pytest
import torch

from test_gpu_evict import IDS, KINDS, check, make, weights

pytestmark = pytest.mark.gpu


def test_filled_length(ctx):
    """In place the cache has at most the budget; another cache keeps the longer of the two."""
    for into_self in (False, True):
        cache = make(torch.bfloat16, 1, 2, 2, 100, 64)
        cache.mark_filled(90)
        cache.evict(90, weights(1, 2, 2, 100, 1, False).cuda(), 40, into=cache if into_self else None)
        assert cache.seq_len() == 40
    cache, other = make(torch.bfloat16, 1, 2, 2, 100, 64), make(torch.bfloat16, 1, 2, 2, 60, 64)
    cache.mark_filled(90)
    for filled, want in ((0, 40), (55, 55)):
        other.mark_filled(filled)
        cache.evict(90, weights(1, 2, 2, 100, 1, False).cuda(), 40, into=other)
        assert cache.seq_len() == 90 and other.seq_len() == want

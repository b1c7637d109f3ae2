"""Eviction from a cache that cannot: refused without a GPU."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv


def test_a_cache_without_sums_neither_observes_nor_evicts():
    cache = kv.MultiLayerPagedKVCache4Bit(1, 16, 64, "cpu", 2, 2, 128)
    assert cache.weights is None
    for call in (lambda: cache.evict(5), lambda: cache.observe(torch.zeros(1, 1, 2, 128), 0)):
        with pytest.raises(RuntimeError, match="track_weights"):
            call()


def test_sums_are_of_every_place_of_the_pages():
    cache = kv.MultiLayerPagedKVCache4Bit(3, 16, 70, "cpu", 2, 4, 128, track_weights=True)
    assert tuple(cache.weights.shape) == (2, 3, 4, 80) and bool((cache.weights == 0).all())
    with pytest.raises(RuntimeError, match="no tokens"):
        cache.evict(5)

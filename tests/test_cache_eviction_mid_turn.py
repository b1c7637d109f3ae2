"""observe and evict where a layer has not had the turn's tokens yet: its last positions are not there, so both are refused (without a GPU: before any launch)."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV


def test_layers_of_different_tokens():
    cache = kv.MultiLayerPagedKVCache4Bit(1, 16, 64, "cpu", 2, 2, 128, track_weights=True)
    cache._needs_init, cache.length, cache._held = [False, False], 21, [21, 20]
    for call in (lambda: cache.evict(5), lambda: cache.observe(torch.zeros(1, 1, 2, 128), 1)):
        with pytest.raises(RuntimeError, match="tokens of this turn"):
            call()
    assert cache.length == 21 and cache.evicted_tokens == 0


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("added", [1, 4])
def test_between_the_layers_of_a_turn(added, f16):
    rows = lambda seed, *shape: torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half().to(DEV)
    cache = kv.MultiLayerPagedKVCache4Bit(2, 16, 128, DEV, 2, 2, 128, disable_quant=f16, track_weights=True)
    for layer in range(2):
        cache.update(rows(layer, 2, 50, 2, 128), rows(layer + 5, 2, 50, 2, 128), layer, {})
        cache.observe(rows(layer + 8, 2, 7, 2, 128), layer)
    for turn in range(2):
        q = rows(20 + turn, 2, added, 2, 128)
        cache.update(rows(21 + turn, 2, added, 2, 128), rows(22 + turn, 2, added, 2, 128), 0, {})(q)
        sums = cache.weights.clone()
        with pytest.raises(RuntimeError, match="tokens of this turn"):
            cache.evict(20)
        with pytest.raises(RuntimeError, match="tokens of this turn"):
            cache.observe(q, 1)
        assert torch.equal(cache.weights, sums)
        cache.observe(q, 0)
        cache.update(rows(23 + turn, 2, added, 2, 128), rows(24 + turn, 2, added, 2, 128), 1, {})(q)
        cache.observe(q, 1)
        cache.evict(20 + turn)
        assert cache.get_seq_length() == 20 + turn

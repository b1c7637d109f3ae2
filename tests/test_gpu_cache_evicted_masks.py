"""Turns with a mask behind an eviction: one of all tokens that there have been is refused and stores nothing, one of those that the cache holds is as none."""
import gc

import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_cache_eviction import rows
from tests.test_gpu_chunk import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_masks_after_an_eviction(window, sinks, f16):
    batch, heads, layers, prompt, keep = 2, 2, 2, 90, 41
    caches = [kv.MultiLayerPagedKVCache4Bit(batch, 16, 128, DEV, layers, heads, 128, disable_quant=f16, window=window, sinks=sinks, track_weights=True) for _ in range(2)]

    def turn(cache, seed, added, mask, layer):
        k, v, q = (rows(seed + 10 * layer + i, batch, added, heads * (2 if i == 2 else 1), 128) for i in range(3))
        return cache.update(k, v, layer, {} if mask is None else {"attention_mask": mask})(q)

    ones = lambda width: torch.ones(batch, width, dtype=torch.int64, device=DEV)
    for cache in caches:
        for layer in range(layers):
            cache.update(rows(layer, batch, prompt, heads, 128), rows(layer + 5, batch, prompt, heads, 128), layer, {"attention_mask": ones(prompt)})
            cache.observe(rows(layer + 8, batch, 30, heads * 2, 128), layer)
        cache.evict(keep, sinks=2, recent=10)
        assert cache.seen_tokens == cache.get_seq_length() == keep and cache.evicted_tokens == prompt - keep
    masked, plain = caches
    for i, added in enumerate([1, 1, 3, 1]):
        held = masked.seen_tokens
        for layer in range(layers):
            now = held + added if layer else held
            before, sums = masked.pages.view(torch.uint8).clone(), masked.weights.clone()
            for width in (held + added + masked.evicted_tokens, held, held + 2 * added):
                with pytest.raises(ValueError, match="attention_mask must be"):
                    turn(masked, 100 * i, added, ones(width), layer)
            left_out = ones(held + added)
            left_out[0, 3] = 0
            with pytest.raises(NotImplementedError, match="evict"):
                turn(masked, 100 * i, added, left_out, layer)
            assert masked.seen_tokens == now and torch.equal(masked.pages.view(torch.uint8), before) and torch.equal(masked.weights, sums)
            o, want = turn(masked, 100 * i, added, ones(held + added), layer), turn(plain, 100 * i, added, None, layer)
            assert torch.equal(o, want) and torch.equal(masked.weights[layer], plain.weights[layer])
    assert masked.seen_tokens == plain.seen_tokens == keep + 6
    masked.evict(20, recent=5)
    assert masked.seen_tokens == 20 and masked.evicted_tokens == prompt + 6 - 20

"""The multi-layer cache without a GPU: turns whose mask says something else than that every sequence brings the new tokens are refused before anything is stored."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv

BATCH, HEADS = 2, 2


def cache_of(held, **kw):
    cache = kv.MultiLayerPagedKVCache4Bit(BATCH, 16, 64, "cpu", 2, HEADS, 128, **kw)
    cache._needs_init, cache.length = [False, False], held
    return cache


def turn(cache, added, mask, layer=0):
    states = torch.zeros(BATCH, added, HEADS, 128, dtype=torch.float16)
    return cache.update(states, states, layer, {"attention_mask": mask})


@pytest.mark.parametrize("disable_quant", [False, True])
@pytest.mark.parametrize("added,window", [(3, 0), (3, 10), (1, 10)])
@pytest.mark.parametrize("layer", [0, 1])
def test_masks_of_later_turns(added, window, layer, disable_quant):
    cache = cache_of(20 if layer == 0 else 20 + added, disable_quant=disable_quant, window=window)
    right = torch.ones(BATCH, 20 + added, dtype=torch.int64)
    for width in (added, 20, 20 + 2 * added):
        with pytest.raises(ValueError, match="attention_mask must be"):
            turn(cache, added, torch.ones(BATCH, width, dtype=torch.int64), layer)
    with pytest.raises(ValueError, match="attention_mask must be"):
        turn(cache, added, right[:1], layer)
    with pytest.raises(ValueError, match="attention_mask must be"):
        turn(cache, added, right[:, None, None], layer)
    short = right.clone()
    short[1, -1] = 0
    with pytest.raises(NotImplementedError, match="padding among the new tokens"):
        turn(cache, added, short, layer)
    cache._padded = True
    with pytest.raises(ValueError, match="padded"):
        turn(cache, added, None, layer)
    assert cache.length == (20 if layer == 0 else 20 + added)


@pytest.mark.parametrize("disable_quant", [False, True])
@pytest.mark.parametrize("window", [0, 10])
def test_a_turn_without_tokens(window, disable_quant):
    cache = cache_of(20, disable_quant=disable_quant, window=window)
    with pytest.raises(AssertionError):
        turn(cache, 0, None)
    assert not cache._pending and cache.length == 20


@pytest.mark.parametrize("disable_quant", [False, True])
@pytest.mark.parametrize("added", [1, 3])
def test_a_refused_turn_leaves_the_length(added, disable_quant):
    """Page counts that differ are refused (kv_cache.py:253-275); the cache holds what it held."""
    cache = cache_of(20, disable_quant=disable_quant)
    mask = torch.ones(BATCH, 20 + added, dtype=torch.int64)
    mask[0, :10] = 0
    with pytest.raises(NotImplementedError, match="different number of pages"):
        turn(cache, added, mask)
    assert cache.length == 20

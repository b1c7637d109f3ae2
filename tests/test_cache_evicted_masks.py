"""The multi-layer cache that tracks weights, without a GPU: a turn of one token whose mask is not of the tokens that the cache holds is refused before anything is stored, as one
of several tokens is.  A generation loop's mask counts the tokens that evict has let go."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_cache_turn_refusals import BATCH, cache_of, turn


@pytest.mark.parametrize("disable_quant", [False, True])
@pytest.mark.parametrize("added", [1, 3])
@pytest.mark.parametrize("layer", [0, 1])
def test_masks_of_other_widths(added, layer, disable_quant):
    held = 20 if layer == 0 else 20 + added
    cache = cache_of(held, disable_quant=disable_quant, track_weights=True)
    assert cache.evicted_tokens == 0
    for gone in (0, 30):
        cache.evicted_tokens = gone
        for width in (20, 20 + added + 30, 20 + added + 1, 1):
            with pytest.raises(ValueError, match="attention_mask must be"):
                turn(cache, added, torch.ones(BATCH, width, dtype=torch.int64), layer)
            assert cache.length == held and not cache._pending


@pytest.mark.parametrize("disable_quant", [False, True])
@pytest.mark.parametrize("added", [1, 3])
def test_masks_that_leave_held_positions_out_after_an_eviction(added, disable_quant):
    """The last columns of a mask say nothing about the positions that stayed."""
    cache = cache_of(20, disable_quant=disable_quant, track_weights=True)
    cache.evicted_tokens = 30
    mask = torch.ones(BATCH, 20 + added, dtype=torch.int64)
    mask[:, 0] = 0
    with pytest.raises(NotImplementedError, match="evict"):
        turn(cache, added, mask)
    assert cache.length == 20


def test_a_padded_prompt_needs_its_mask():
    cache = cache_of(20, track_weights=True)
    cache._padded = True
    with pytest.raises(ValueError, match="padded"):
        turn(cache, 1, None)

"""Turns of several tokens behind a padded prompt: every sequence's own length counts (two pages each: the class asks for one page count)."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, definition
from tests.test_gpu_chunk_cache import rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (12, 2)])
def test_turns_behind_a_padded_prompt(window, sinks, f16):
    batch, heads, group, prompt, layers = 2, 2, 3, 30, 2
    cache = kv.MultiLayerPagedKVCache4Bit(batch, 16, 64, DEV, layers, heads, 128, disable_quant=f16, hadamard_dtype=None, window=window, sinks=sinks)
    mask = torch.ones(batch, prompt, dtype=torch.int64, device=DEV)
    mask[0, :5], mask[1, :12] = 0, 0
    for layer in range(layers):
        cache.update(rows(layer, batch, prompt, heads, 128), rows(layer + 5, batch, prompt, heads, 128), layer, {"attention_mask": mask})
    for turn, added in enumerate([3, 1, 3]):
        mask = torch.cat([mask, mask.new_ones(batch, added)], dim=1)
        lens = mask.sum(1).tolist()
        for layer in range(layers):
            k, v, q = (rows(100 * turn + 10 * layer + i, batch, added, heads * (group if i == 2 else 1), 128) for i in range(3))
            if added > 1 or window:                         # (refused; nothing is stored, unused entries may be anything)
                before, held = cache.pages.view(torch.uint8).clone(), cache.get_seq_length()
                with pytest.raises(ValueError, match="padded"):
                    cache.update(k, v, layer, {})
                assert torch.equal(cache.pages.view(torch.uint8), before) and cache.get_seq_length() == held
            o = cache.update(k, v, layer, {"attention_mask": mask})(q)
            specs = cache.get_cache_specs_for_flash_infer(mask)
            want, tol = definition(specs, q.reshape(-1, heads * group, 128), lens, [added] * batch, layer, window, sinks)
            assert bool(((o.double().reshape(want.shape) - want).abs() <= tol).all()), (turn, layer)
            if f16:
                for b in range(batch):
                    for i in range(added):
                        pos = lens[b] - added + i
                        assert torch.equal(cache.pages[pos // 16 * batch + b, layer, 0, :, pos % 16], k[b, i])

"""The multi-layer cache that keeps track of attention weights and evicts by them: its sums and its attention are those of the entry points, against their definitions in
64 bits (test_gpu_evict.py, test_gpu_chunk.py, with their tolerances), before and after positions go."""
import gc
import math

import numpy as np
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV
from tests.test_gpu_chunk import definition as attention
from tests.test_gpu_evict import bits, logarithms, stays
from tests.test_gpu_evict import definition as weights_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def rows(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).half().to(DEV)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("group,window,sinks", [(1, 0, 0), (4, 0, 0), (2, 60, 4)])
def test_turns_sums_and_evictions(group, window, sinks, f16):
    batch, heads, layers, prompt = 2, 2, 2, 150
    cache = kv.MultiLayerPagedKVCache4Bit(batch, 16, 400, DEV, layers, heads, 128, disable_quant=f16, hadamard_dtype=None, window=window, sinks=sinks, track_weights=True)
    want = torch.zeros(cache.weights.shape, dtype=torch.float64, device=DEV)
    off = torch.zeros_like(want)

    def turn(seed, added, first=False):
        for layer in range(layers):
            out = cache.update(rows(seed + layer, batch, added, heads, 128), rows(seed + layer + 50, batch, added, heads, 128), layer, {})
            asking = min(added, 64)
            q = rows(seed + layer + 70, batch, asking, heads * group, 128)
            o = cache.observe(q, layer) if first else out(q)
            assert o.shape == q.shape
            specs, length = cache.get_cache_specs_for_flash_infer(None), cache.get_seq_length()
            flat, lens, news = q.reshape(-1, heads * group, 128), [length] * batch, [asking] * batch
            right, tol = attention(specs, flat, lens, news, layer, window, sinks)
            assert bool(((o.double().reshape(right.shape) - right).abs() <= tol).all()), (seed, layer)
            lse = logarithms(specs, flat, lens, news, layer, window, sinks)
            more, tol = weights_of(specs, flat, lse, torch.zeros(batch, heads, want.shape[3], device=DEV), lens, news, layer, window, sinks)
            # (the attention's own logarithms are those of rounded weights: within 2^-11, and what its logits' errors add; see test_gpu_shared.py)
            want[layer] += more
            off[layer] += tol + 2.0 ** -10 * more + 2.0 ** -23 * want[layer]
            assert bool(((cache.weights[layer].double() - want[layer]).abs() <= off[layer]).all()), (seed, layer)

    turn(0, prompt, first=True)
    for k, added in enumerate([1, 1, 5, 30]):
        turn(100 * (k + 1), added)
    for k, (keep, first, recent) in enumerate([(100, 4, 20), (60, 0, 60), (33, 1, 8)]):
        held = cache.get_seq_length()
        specs = {name: t.clone() for name, t in cache.get_cache_specs_for_flash_infer(None).items()}
        sums = cache.weights.clone()
        cache.evict(keep, sinks=first, recent=recent)
        assert cache.get_seq_length() == min(held, keep)
        at = specs["kv_indices"].view(batch, -1).long()
        for layer in range(layers):
            kept, _ = stays(sums[layer].cpu().numpy(), np.full(batch, held), keep, first, recent)
            for b in range(batch):
                for h in range(heads):
                    s, t = torch.from_numpy(kept[b, h]).long().to(DEV), torch.arange(keep, device=DEV)
                    for name, now in (("kv_data", cache.pages), ("kv_param", cache.scales)):
                        assert torch.equal(bits(now)[at[b][t // 16], layer, :, h, t % 16], bits(specs[name])[at[b][s // 16], layer, :, h, s % 16])
                    assert torch.equal(cache.weights[layer, b, h, :keep], sums[layer, b, h, s]) and bool((cache.weights[layer, b, h, keep:] == 0).all())
        want.copy_(cache.weights), off.copy_(2.0 ** -23 * want)
        cache.evict(keep + 1)                               # (nothing to do)
        assert cache.get_seq_length() == min(held, keep)
        turn(1000 * (k + 1), 7)
        turn(1000 * (k + 1) + 500, 1)


@pytest.mark.parametrize("f16", [False, True])
def test_the_transform_of_keys_and_queries(f16):
    """hadamard_dtype fp16: the sums go with the transformed keys, each row's add up to its query heads."""
    cache = kv.MultiLayerPagedKVCache4Bit(1, 16, 200, DEV, 1, 2, 128, disable_quant=f16, track_weights=True)
    cache.update(rows(1, 1, 90, 2, 128), rows(2, 1, 90, 2, 128), 0, {})
    cache.observe(rows(3, 1, 30, 8, 128), 0)
    for k in range(3):
        cache.update(rows(4 + k, 1, 1, 2, 128), rows(14 + k, 1, 1, 2, 128), 0, {})(rows(24 + k, 1, 1, 8, 128))
    assert bool(((cache.weights.double().sum(-1) - 33 * 4).abs() <= 33 * 4 * 2.0 ** -10).all())
    cache.evict(40, sinks=2, recent=10)
    assert cache.get_seq_length() == 40 and bool((cache.weights[..., 40:] == 0).all())


def test_a_cache_that_does_not_track_is_as_before():
    outs = []
    for track in (False, True):
        cache = kv.MultiLayerPagedKVCache4Bit(2, 16, 128, DEV, 1, 2, 128, track_weights=track)
        cache.update(rows(1, 2, 50, 2, 128), rows(2, 2, 50, 2, 128), 0, {})
        outs.append(cache.update(rows(3, 2, 1, 2, 128), rows(4, 2, 1, 2, 128), 0, {})(rows(5, 2, 1, 2, 128)))
        assert (cache.weights is None) == (not track)
    assert torch.allclose(*outs, rtol=4e-3, atol=4e-3)      # (the step without sums is the decode kernel's)


def test_refusals():
    cache = kv.MultiLayerPagedKVCache4Bit(2, 16, 128, DEV, 2, 2, 128, track_weights=True)
    with pytest.raises(RuntimeError, match="no tokens"):
        cache.evict(10)
    cache.update(rows(1, 2, 50, 2, 128), rows(2, 2, 50, 2, 128), 0, {})
    with pytest.raises(RuntimeError, match="no tokens"):
        cache.evict(10)
    with pytest.raises(RuntimeError, match="no tokens"):
        cache.observe(rows(3, 2, 1, 2, 128), 1)
    cache.observe(rows(3, 2, 1, 2, 128), 0)
    for q in (rows(3, 1, 1, 2, 128), rows(3, 2, 51, 2, 128), rows(3, 2, 0, 2, 128)):
        with pytest.raises(ValueError):
            cache.observe(q, 0)
    cache.update(rows(1, 2, 50, 2, 128), rows(2, 2, 50, 2, 128), 1, {})
    for bad in ({"keep": 0}, {"keep": 10, "sinks": 6, "recent": 5}, {"keep": 10, "sinks": -1}, {"keep": 10, "recent": -1}):
        with pytest.raises(ValueError):
            cache.evict(**bad)
    assert cache.get_seq_length() == 50
    mask = torch.ones(2, 50, dtype=torch.int64, device=DEV)
    mask[1, :1] = 0                                         # (as many pages as the other sequence, which the class needs)
    padded = kv.MultiLayerPagedKVCache4Bit(2, 16, 128, DEV, 1, 2, 128, track_weights=True)
    padded.update(rows(1, 2, 50, 2, 128), rows(2, 2, 50, 2, 128), 0, {"attention_mask": mask})
    with pytest.raises(NotImplementedError):
        padded.evict(10)
    with pytest.raises(NotImplementedError):
        padded.observe(rows(3, 2, 1, 2, 128), 0)

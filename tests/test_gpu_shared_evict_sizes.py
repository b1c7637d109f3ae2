"""Shared prefixes and eviction where sizes are large: pools and sums beyond 32-bit offsets, batches and lists beyond one workgroup's or one launch's share."""
import gc

import numpy as np
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, make
from tests.test_gpu_evict import bits, check, random_lists, stays
from tests.test_gpu_shared import check as check_shared
from tests.test_gpu_shared import make_shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[250, 6], [1, 1]])
def test_pages_beyond_32_bit_offsets(news, f16):
    """A pool of more than 2^32 bytes, its last pages in use: the same bits as from a small one."""
    lens, prefixes = [600, 90], [200]
    specs, prefix, q, starts = make_shared(5, 16, prefixes, None, lens, news, 28, 8, f16, spare=0)
    per, data = specs["kv_data"].shape[0], specs["kv_data"]
    total = (5 << 30) // (data[0].numel() * data.element_size())
    pool = {name: torch.empty((total, *specs[name].shape[1:]), dtype=specs[name].dtype, device=DEV) for name in ("kv_data", "kv_param")}
    for name, t in pool.items():
        t[total - per:] = specs[name]
    assert pool["kv_data"].numel() * data.element_size() > 1 << 32
    far = {**specs, **pool, "kv_indices": specs["kv_indices"] + (total - per)}
    pick = lambda name: getattr(kv, name + ("_f16" if f16 else "_i4"))
    results = []
    for used in (specs, far):
        o, lse, sums = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV), torch.zeros(2, 28, 600, device=DEV)
        pick("batch_shared")(o, q, **used, layer_idx=1, **{**prefix, "prefix_indices": used["kv_indices"]}, seqlen_indptr=starts, lse=lse)
        pick("accumulate_weights")(sums, q, lse, **used, layer_idx=1, seqlen_indptr=starts)
        kept, _ = kv.heavy_positions(sums, torch.tensor(lens, dtype=torch.int32, device=DEV), 77, sinks=2, recent=20)
        pick("keep_positions")(kept, **used, layer_idx=1, weights=sums)
        results.append([o, lse, sums, kept, bits(used["kv_data"][-per:]), bits(used["kv_param"][-per:])])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_sums_beyond_32_bit_offsets():
    """Sums of more than 2^32 bytes: the last sequence's are added to, gone through and moved."""
    batch, heads, capacity, n = 9, 2, 1 << 26, 5000
    weights = torch.zeros(batch, heads, capacity, device=DEV)
    assert weights.numel() * 4 > 1 << 32
    lens = [20] * (batch - 1) + [n]
    specs, q, starts = make(2, 16, lens, [1] * batch, heads, 4, spare=0)
    lse = torch.full(q.shape[:2], 3.0, device=DEV)
    kv.accumulate_weights_i4(weights, q, lse, **specs, layer_idx=1, max_seq_len=n)
    small = torch.zeros(batch, heads, n, device=DEV)
    kv.accumulate_weights_i4(small, q, lse, **specs, layer_idx=1, max_seq_len=n)
    assert torch.equal(weights[..., :n], small) and float(small[-1].min()) > 0
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept, left = kv.heavy_positions(weights, lengths, 1000, sinks=4, recent=100)
    want, new = stays(small.cpu().numpy(), np.asarray(lens), 1000, 4, 100)
    assert torch.equal(kept.cpu(), torch.from_numpy(want)) and left.tolist() == new.tolist()
    kv.keep_positions_i4(kept, **specs, layer_idx=1, weights=weights)
    kv.keep_positions_i4(kept, **specs, layer_idx=0, weights=small)
    assert torch.equal(weights[..., :n], small)


@pytest.mark.parametrize("f16", [False, True])
def test_large_batches(f16):
    """Sequences beyond those whose work items are counted, most without many tokens; prefixes of many of them."""
    batch, prefixes = 300, 40
    news = [(7 * b) % 4 for b in range(batch)]
    lens = [n + (13 * b) % 20 for b, n in enumerate(news)]
    members = sorted((29 * p) % (batch + 1) for p in range(prefixes + 1))
    specs, prefix, q, starts = make_shared(3, 16, [(11 * p) % 70 for p in range(prefixes)], members, lens, news, 2, 4, f16)
    check_shared(specs, prefix, q, starts, [(11 * p) % 70 for p in range(prefixes)], members, lens, news)
    check(specs, q, starts, lens, news)
    kept = random_lists(1, lens, 2, 9)
    before = [bits(specs[name]).clone() for name in ("kv_data", "kv_param")]
    (kv.keep_positions_f16 if f16 else kv.keep_positions_i4)(kept, **specs, layer_idx=0)
    bounds, pages = specs["kv_indptr"].tolist(), specs["kv_indices"].long()
    for b in range(0, batch, 7):
        n = min(9, lens[b])
        table, source, to = pages[bounds[b]:bounds[b + 1]], kept[b, 1, :n].long(), torch.arange(n, device=DEV)
        for old, name in zip(before, ("kv_data", "kv_param")):
            if n:
                assert torch.equal(bits(specs[name])[table[to // 16], 0, :, 1, to % 16], old[table[source // 16], 0, :, 1, source % 16])


@pytest.mark.parametrize("batch,heads", [(1, 1), (70000, 1)])
def test_many_lists(batch, heads):
    g = torch.Generator().manual_seed(batch)
    weights = torch.rand(batch, heads, 12, generator=g)
    lengths = torch.randint(0, 13, (batch,), generator=g).int()
    kept, left = kv.heavy_positions(weights.to(DEV), lengths.to(DEV), 5, sinks=1, recent=1)
    place = torch.arange(12)
    rank = torch.where((place < 1) | (place >= lengths[:, None] - 1), 2.0, weights[:, 0])
    rank = torch.where(place < lengths[:, None], rank, -1.0)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :5]
    count = lengths.clamp(max=5)[:, None]
    order = torch.where(torch.arange(5) < count, order, 99).sort(-1).values
    assert torch.equal(kept[:, 0].cpu().long(), torch.where(order == 99, -1, order)) and torch.equal(left.cpu(), lengths.clamp(max=5))

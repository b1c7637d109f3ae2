"""Shared prefixes and eviction: the native route and the one in Python give the same bits and raise the same errors; caches whose sizes nothing could be computed for come back as
errors on both."""
import pytest
import torch

from quarot_amd import _lib
from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, make
from tests.test_gpu_shared import make_shared

pytestmark = pytest.mark.gpu
NAMES = ("chunk", "shared", "accumulate", "heavy_positions", "keep_positions")


@pytest.fixture(params=[True, False], ids=["native", "python"])
def route(request, monkeypatch):
    if not request.param:
        for name in NAMES:
            monkeypatch.setattr(_lib.host, name, lambda *a: None)


def everything(f16, step):
    lens, news, prefixes = [90, 33], [1, 1] if step else [30, 5], [70]
    specs, prefix, q, starts = make_shared(1, 16, prefixes, None, lens, news, 2, 4, f16, fused=256)
    pick = lambda name: getattr(kv, name + ("_f16" if f16 else "_i4"))
    o, lse = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape[:2], device=DEV)
    bounds = None if step else starts
    pick("batch_shared")(o, q, **specs, layer_idx=1, **prefix, seqlen_indptr=bounds, lse=lse, max_seq_len=90, max_prefix_len=70)
    alone, own = torch.empty_like(o), torch.empty_like(lse)
    pick("batch_chunk")(alone, q, **specs, layer_idx=1, seqlen_indptr=bounds, lse=own)
    sums = torch.zeros(2, 2, 100, device=DEV)
    pick("accumulate_weights")(sums, q, lse, **specs, layer_idx=1, seqlen_indptr=bounds)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    kept, left = kv.heavy_positions(sums, lengths, 20, sinks=2, recent=5)
    before = sums.clone()
    pick("keep_positions")(kept, **specs, layer_idx=1, weights=sums)
    return [o, lse, alone, own, before, kept, left, sums, specs["kv_data"][..., :64].clone().nan_to_num() if f16 else specs["kv_data"].clone()]


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("f16", [False, True])
def test_both_routes_give_the_same_bits(f16, step, monkeypatch):
    native = everything(f16, step)
    called = []
    for name in NAMES:
        monkeypatch.setattr(_lib.host, name, lambda *a, name=name: called.append(name))
    for a, b in zip(native, everything(f16, step)):
        assert torch.equal(a, b)
    assert set(NAMES[1:]) <= set(called)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("axis,match", [(3, "multiple|kept|weights"), (4, "invalid size"), (0, "invalid size"), (1, "layer_idx")])
def test_caches_without_heads_entries_pages_or_layers(axis, match, f16, route):
    specs, prefix, q, starts = make_shared(1, 16, [7], None, [20, 5], [3, 2], 2, 2, f16)
    empty = {**specs, **{name: specs[name].narrow(axis, 0, 0).contiguous() for name in ("kv_data", "kv_param")}}
    pick = lambda name: getattr(kv, name + ("_f16" if f16 else "_i4"))
    o, lse, sums = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.zeros(q.shape[:2], device=DEV), torch.zeros(2, 2, 20, device=DEV)
    kept = torch.zeros(2, 2, 3, dtype=torch.int32, device=DEV)
    for call in (lambda: pick("batch_shared")(o, q, **empty, layer_idx=0, **prefix, seqlen_indptr=starts), lambda: pick("accumulate_weights")(sums, q, lse, **empty, layer_idx=0, seqlen_indptr=starts),
                 lambda: pick("keep_positions")(kept, **empty, layer_idx=0, weights=sums)):
        with pytest.raises(RuntimeError, match=match):
            call()


def test_refusals_on_both_routes(route):
    from tests import test_gpu_evict, test_gpu_shared
    test_gpu_shared.test_refusals()
    test_gpu_evict.test_refusals()


def test_on_another_stream_than_the_current_one(route):
    """Everything goes to torch's current stream: work there is in order without waiting for the device."""
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        first = everything(False, False)
    stream.synchronize()
    for a, b in zip(first, everything(False, False)):
        assert torch.equal(a, b)


def test_a_prefix_of_unknown_length_is_cut_by_its_page_list(monkeypatch):
    """Without a largest length the launch is sized for what the page list has room for, on both routes: the bits of a call that gives that number."""
    specs, prefix, q, starts = make_shared(2, 16, [3000], None, [90, 33], [1, 1], 2, 4)
    room = prefix["prefix_indices"].shape[0] * 16

    def run(**hint):
        o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        kv.batch_shared_i4(o, q, **specs, layer_idx=1, **prefix, seqlen_indptr=starts, **hint)
        return o

    native = run()
    assert torch.equal(native, run(max_prefix_len=room))
    monkeypatch.setattr(_lib.host, "shared", lambda *a: None)
    assert torch.equal(native, run()) and torch.equal(native, run(max_prefix_len=room))

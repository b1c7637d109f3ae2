"""The multi-layer cache with more than one new token, with a window, and with grouped query heads: its pages are those of the entry points, its attention is
batch_chunk_i4's and batch_chunk_f16's, against the definition in 64 bits (test_gpu_chunk.py, with its tolerances)."""
import gc

import pytest
import torch

from quarot_amd import _lib
from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, check, definition, make

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


def specs_of(cache):
    specs = cache.get_cache_specs_for_flash_infer(None)
    cache.pages                                             # (a held token is stored)
    return specs


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("group,window,sinks", [(1, 0, 0), (4, 0, 0), (3, 20, 4), (1, 7, 0)])
def test_turns_of_several_tokens(group, window, sinks, f16):
    batch, heads, prompt, layers = 2, 2, 37, 2
    cache = kv.MultiLayerPagedKVCache4Bit(batch, 16, 128, DEV, layers, heads, 128, disable_quant=f16, hadamard_dtype=None, window=window, sinks=sinks)
    stored = [[], []]
    for turn, added in enumerate([prompt, 5, 1, 1, 40]):
        for layer in range(layers):
            k, v = rows(100 * turn + layer, batch, added, heads, 128), rows(100 * turn + layer + 50, batch, added, heads, 128)
            stored[layer].append((k, v))
            out = cache.update(k, v, layer, {})
            if turn == 0:
                assert out[0] is k and out[1] is v
                continue
            q = rows(100 * turn + layer + 70, batch, added, heads * group, 128)
            o = out(q)
            assert o.shape == q.shape and o.dtype == torch.float16
            specs, length = specs_of(cache), cache.get_seq_length()
            want, tol = definition(specs, q.reshape(-1, heads * group, 128), [length] * batch, [added] * batch, layer, window, sinks)
            if group == 1 and added == 1 and not window:    # (the step without a window is batch_decode's, which rounds more)
                assert torch.allclose(o.reshape(want.shape), want.half(), rtol=4e-3, atol=4e-3)
            else:
                assert bool(((o.double().reshape(want.shape) - want).abs() <= tol).all()), (turn, layer)
    # all the tokens in one piece give the same pages
    other = kv.MultiLayerPagedKVCache4Bit(batch, 16, 128, DEV, layers, heads, 128, disable_quant=f16, hadamard_dtype=None)
    for layer in range(layers):
        other.update(*(torch.cat([t[side] for t in stored[layer]], dim=1) for side in (0, 1)), layer, {})
    length = other.get_seq_length()
    assert length == cache.get_seq_length() == 84
    for pos in range(length):
        for b in range(batch):
            page = pos // 16 * batch + b
            assert torch.equal(cache.pages[page, :, :, :, pos % 16], other.pages[page, :, :, :, pos % 16])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_queries_are_transformed_like_keys(dtype, f16):
    """With the Hadamard transform over keys and queries attention is what it is without one, up to the rounding of both."""
    batch, heads, group, prompt, added = 2, 2, 2, 30, 6
    plain, turned = (kv.MultiLayerPagedKVCache4Bit(batch, 16, 64, DEV, 1, heads, 128, disable_quant=True, hadamard_dtype=h) for h in (None, dtype))
    coded = turned if f16 else kv.MultiLayerPagedKVCache4Bit(batch, 16, 64, DEV, 1, heads, 128, hadamard_dtype=dtype)
    outs = []
    q = rows(3, batch, added, heads * group, 128)
    for cache in (plain, coded):
        cache.update(rows(1, batch, prompt, heads, 128), rows(2, batch, prompt, heads, 128), 0, {})
        outs.append(cache.update(rows(4, batch, added, heads, 128), rows(5, batch, added, heads, 128), 0, {})(q).double())
    off = float((outs[0] - outs[1]).norm() / outs[0].norm())
    # fp16 pages: q and k are rounded to fp16 once more each, 2^-11 at most of their elements; 4-bit codes: half a step of a range of about 5 in 15, sqrt(1 / 12) of it
    # per element of a value of unit size, and as much for the logits
    assert off < (2.0 ** -9 if f16 else 2 * 5 / 15 / 12 ** 0.5 * 1.5), off


def test_several_tokens_after_single_ones_and_refusals():
    cache = kv.MultiLayerPagedKVCache4Bit(1, 16, 64, DEV, 1, 2, 128)
    one = lambda n, h=2: rows(9, 1, n, h, 128)
    cache.update(one(10), one(10), 0, {})
    step = cache.update(one(1), one(1), 0, {})              # its token is held for the call
    with pytest.raises(AssertionError):
        step(one(2))
    more = cache.update(one(3), one(3), 0, {})              # stores it
    assert more(one(3, 6)).shape == (1, 3, 6, 128)
    with pytest.raises(AssertionError):
        more(one(1))
    with pytest.raises(RuntimeError, match="multiple"):
        more(one(3, 3))
    grouped = cache.update(one(1), one(1), 0, {})
    assert grouped(one(1, 4)).shape == (1, 1, 4, 128) and not cache._pending
    with pytest.raises(NotImplementedError):
        cache.update(one(60), one(60), 0, {})
    for bad in ({"window": -1}, {"sinks": -1}):
        with pytest.raises(ValueError):
            kv.MultiLayerPagedKVCache4Bit(1, 16, 64, DEV, 1, 2, 128, **bad)


def test_turn_captured_and_replayed():
    """A turn's update and attention in a graph, replayed with other tokens."""
    cache = kv.MultiLayerPagedKVCache4Bit(1, 16, 256, DEV, 1, 2, 128, window=50, sinks=2)
    k, v, q = rows(1, 1, 20, 2, 128), rows(2, 1, 20, 2, 128), rows(3, 1, 20, 8, 128)
    cache.update(rows(4, 1, 100, 2, 128), rows(5, 1, 100, 2, 128), 0, {})
    eager = cache.update(k, v, 0, {})(q).clone()
    cache.length -= 20
    cache._specs = None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = cache.update(k, v, 0, {})(q)
    for turn in range(3):
        graph.replay()
        torch.cuda.synchronize()
        if turn == 0:
            assert torch.equal(out, eager)
        specs = specs_of(cache)
        want = torch.empty(20, 8, 128, dtype=torch.float16, device=DEV)
        kv.batch_chunk_i4(want, q[0], **{n: specs[n] for n in specs}, layer_idx=0, seqlen_indptr=torch.tensor([0, 20], dtype=torch.int32, device=DEV),
                          max_new_len=20, max_seq_len=120, window=50, sinks=2, q_hadamard=True)
        assert torch.equal(out[0], want), turn
        k.copy_(rows(10 + turn, 1, 20, 2, 128)), v.copy_(rows(20 + turn, 1, 20, 2, 128)), q.copy_(rows(30 + turn, 1, 20, 8, 128))


@pytest.fixture
def large_memory():
    """What the test allocates goes back to the device behind it (a later test fills the memory up to a limit)."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("new", [4, 40, 300])
@pytest.mark.parametrize("f16", [False, True])
def test_pages_beyond_32_bit_offsets(new, f16, large_memory):
    """A pool of more than 2^32 bytes, its last pages in use."""
    specs, q, starts = make(5, 16, [500, 310], [new, 2], 8, 1, f16, layers=2, spare=0)
    per = specs["kv_data"].shape[0]
    bytes_per = specs["kv_data"][0].numel() * specs["kv_data"].element_size()
    total = (5 << 30) // bytes_per
    data = torch.empty((total, *specs["kv_data"].shape[1:]), dtype=specs["kv_data"].dtype, device=DEV)
    param = torch.empty((total, *specs["kv_param"].shape[1:]), dtype=torch.float16, device=DEV)
    data[total - per:], param[total - per:] = specs["kv_data"], specs["kv_param"]
    assert data.numel() * data.element_size() > 1 << 32
    outs = [torch.empty_like(q) for _ in range(2)]
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    call(outs[0], q, **specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=500)
    call(outs[1], q, **{**specs, "kv_data": data, "kv_param": param, "kv_indices": specs["kv_indices"] + (total - per)}, layer_idx=1, seqlen_indptr=starts,
         max_new_len=new, max_seq_len=500)
    assert torch.equal(*outs)


@pytest.mark.parametrize("f16", [False, True])
def test_without_the_native_host_side(f16, monkeypatch):
    """The call in Python is the native one, to the bit; tables too."""
    specs, q, starts = make(8, 16, [300, 70], [30, 7], 2, 4, f16)
    native, = check(specs, q, starts, [300, 70], [30, 7], hints=(True,))
    lengths, news = (torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([300, 70], [30, 7]))
    tables = kv.build_page_tables(lengths, 16, 20, new_lengths=news, tokens=40)
    monkeypatch.setattr(_lib.host, "chunk", lambda *a: None)
    monkeypatch.setattr(_lib.host, "build_page_tables", lambda *a: None)
    plain, = check(specs, q, starts, [300, 70], [30, 7], hints=(True,))
    assert torch.equal(native, plain)
    other = kv.build_page_tables(lengths, 16, 20, new_lengths=news, tokens=40)
    assert list(other) == list(tables) and all(torch.equal(tables[n], other[n]) for n in tables)

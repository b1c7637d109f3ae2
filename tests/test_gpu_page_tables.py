"""build_page_tables: whole numbers, equal to a loop over the sequences on the CPU."""
import gc

import pytest
import torch

from quarot_amd.transformers import kv_cache as kv

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def by_hand(lengths, page_size, max_pages, table, new, tokens):
    batch = len(lengths)
    lengths = [min(max(n, 0), max_pages * page_size) for n in lengths]
    indptr, indices, last, starts, positions, slots = [0], [], [], [0], [], []
    for b, n in enumerate(lengths):
        pages = -(-n // page_size)
        number = [table[b][i] if table is not None else i * batch + b for i in range(max_pages)]
        indices += number[:pages]
        indptr.append(len(indices))
        last.append(n - (pages - 1) * page_size if n else 0)
        if new is not None:
            fresh = max(new[b], 0)
            starts.append(starts[-1] + fresh)
            for p in range(n - fresh, n):
                positions.append(p)
                slots.append(number[p // page_size] * page_size + p % page_size if p >= 0 and number[p // page_size] >= 0 else -1)
    indices += [-1] * (batch * max_pages - len(indices))
    pad = [-1] * max(0, tokens - len(positions))
    return indptr, indices, last, starts, (positions + pad)[:tokens], (slots + pad)[:tokens]


@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("page_size", [16, 1, 7, 128])
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([0], [0]), ([16, 17, 0, 33], [16, 1, 0, 2]), ([5, 500, 64], None), ([5, 500, 64], [7, 500, 0]),
                                         (list(range(300)), [i % 3 for i in range(300)]), ([100000], [3000]), ([-4, 20], [2, -1])])
def test_tables_and_slots(lengths, new, page_size, table):
    g = torch.Generator().manual_seed(page_size)
    batch, width = len(lengths), max(1, max(-(-n // page_size) for n in lengths)) + 2
    rows = torch.randint(-1, 1 << 20, (batch, width + 3), generator=g, dtype=torch.int32) if table else None
    tokens = 0 if new is None else sum(max(n, 0) for n in new)
    for asked in {tokens, tokens + 5, max(0, tokens - 1)} if new is not None else {0}:
        got = kv.build_page_tables(torch.tensor(lengths, dtype=torch.int32, device=DEV), page_size, width,
                                   block_table=None if rows is None else rows.to(DEV)[:, :width],
                                   new_lengths=None if new is None else torch.tensor(new, dtype=torch.int32, device=DEV), tokens=asked)
        want = by_hand(lengths, page_size, width, None if rows is None else rows.tolist(), new, asked)
        names = ("kv_indptr", "kv_indices", "last_page_offset") + (("seqlen_indptr", "positions", "slots") if new is not None else ())
        assert sorted(got) == sorted(names)
        for name, w in zip(names, want):
            assert got[name].dtype == (torch.int64 if name in ("positions", "slots") else torch.int32)
            assert got[name].tolist() == w, name


def test_lengths_beyond_the_table_and_one_common_length():
    """A length beyond max_pages * page_size counts as that; a common length gives qr_page_tables' tables."""
    got = kv.build_page_tables(torch.tensor([100, 20], dtype=torch.int32, device=DEV), 16, 2, new_lengths=torch.tensor([3, 1], dtype=torch.int32, device=DEV),
                               tokens=4)
    want = by_hand([100, 20], 16, 2, None, [3, 1], 4)
    for name, w in zip(("kv_indptr", "kv_indices", "last_page_offset", "seqlen_indptr", "positions", "slots"), want):
        assert got[name].tolist() == w
    cache = kv.MultiLayerPagedKVCache4Bit(3, 16, 100, DEV, 1, 2, 128)
    cache.length = 70
    specs = cache.get_cache_specs_for_flash_infer(None)
    got = kv.build_page_tables(torch.full((3,), 70, dtype=torch.int32, device=DEV), 16, 7)
    for name in ("kv_indptr", "last_page_offset"):
        assert torch.equal(got[name], specs[name])
    assert torch.equal(got["kv_indices"][:15], specs["kv_indices"]) and bool((got["kv_indices"][15:] == -1).all())


def test_captured_and_replayed_with_other_lengths():
    lengths, new = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([40, 7], [2, 3]))
    kv.build_page_tables(lengths, 16, 8, new_lengths=new, tokens=5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv.build_page_tables(lengths, 16, 8, new_lengths=new, tokens=5)
    for values in ([40, 7], [100, 90], [3, 16], [40, 7]):
        lengths.copy_(torch.tensor(values, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for name, w in zip(("kv_indptr", "kv_indices", "last_page_offset", "seqlen_indptr", "positions", "slots"), by_hand(values, 16, 8, None, [2, 3], 5)):
            assert got[name].tolist() == w


def test_tables_drive_append_and_attention():
    """Lengths on the GPU -> tables -> quantise and append -> attention, for sequences with unequal page counts, against separate caches of each."""
    heads, page, lens, news = 2, 16, [40, 100, 3], [40, 17, 1]
    lengths, fresh = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (lens, news))
    t = kv.build_page_tables(lengths, page, 7, new_lengths=fresh, tokens=sum(news))
    g = torch.Generator(device=DEV).manual_seed(1)
    pool = {"kv_data": torch.randint(0, 256, (21, 1, 2, heads, page, 64), generator=g, device=DEV, dtype=torch.uint8),
            "kv_param": torch.rand(21, 1, 2, heads, page, 2, generator=g, device=DEV).half()}
    specs = {**pool, **{k: t[k] for k in ("kv_indptr", "kv_indices", "last_page_offset")}}
    q, k, v = (torch.randn(sum(news), heads, 128, generator=g, device=DEV).half() for _ in range(3))
    kv.quantize_append_kv_i4(**specs, k=k, v=v, seqlen_indptr=t["seqlen_indptr"], layer_idx=0)
    o = torch.empty_like(q)
    kv.batch_chunk_i4(o, q, **specs, layer_idx=0, seqlen_indptr=t["seqlen_indptr"])
    codes, scale, zero = kv.asym_quantize_and_pack_i4(v)
    flat = pool["kv_data"].permute(0, 4, 1, 2, 3, 5).reshape(21 * page, 2, heads, 64)       # slot -> its vectors
    assert torch.equal(flat[t["slots"], 1], codes)
    at = 0
    for b in range(3):
        alone = {**pool, "kv_indptr": t["kv_indptr"][b:b + 2] - t["kv_indptr"][b], "kv_indices": t["kv_indices"][int(t["kv_indptr"][b]):],
                 "last_page_offset": t["last_page_offset"][b:b + 1]}
        one = torch.empty_like(q[at:at + news[b]])
        kv.batch_chunk_i4(one, q[at:at + news[b]], **alone, layer_idx=0, seqlen_indptr=torch.tensor([0, news[b]], dtype=torch.int32, device=DEV))
        assert torch.equal(one, o[at:at + news[b]])
        at += news[b]


def test_refusals():
    n = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    for match, args, kw in (("int32", (n.long(), 16, 2), {}), ("CUDA", (n.cpu(), 16, 2), {}), ("positive", (n, 0, 2), {}), ("positive", (n, 16, 0), {}),
                            ("needed", (n, 16), {}), ("without", (n, 16, 2), {"tokens": 3}), ("new_lengths", (n, 16, 2), {"new_lengths": n[:1]}),
                            ("block_table", (n, 16, 2), {"block_table": n}), ("columns", (n, 16, 4), {"block_table": torch.zeros(2, 3, dtype=torch.int32, device=DEV)}),
                            ("positive", (n, 16, 2), {"new_lengths": n, "tokens": -1})):
        with pytest.raises(RuntimeError, match=match):
            kv.build_page_tables(*args, **kw)
    with pytest.raises(RuntimeError, match="invalid size"):
        kv.build_page_tables(n, 16, 1 << 30)
    none = kv.build_page_tables(n[:0], 16, 2, new_lengths=n[:0], tokens=2)
    assert none["kv_indptr"].tolist() == [0] and none["seqlen_indptr"].tolist() == [0] and none["slots"].tolist() == [-1, -1]

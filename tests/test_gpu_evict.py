"""Eviction from the paged cache: accumulated attention weights against their definition in 64 bits, the positions that stay and their move exactly, and a run of
them together, as they are used.

How far a position's sum may be off, with s_r its logit against row r, p_r = exp(s_r - lse_r) and half a step of fp32 being 2^-24: every p_r by p_r times
  140 * 2^-24 * (the logit's absolute terms)          its product in fp32 (128 products and a few more operations)
  2^-21 (1 + |s_r| + |lse_r|)                          the exponential's argument, base 2, and the exponential itself
and the sum by 256 additions' roundings of it (rows are added up in blocks, blocks in 32 bits): 2^-16 of what it holds.  Nothing is rounded to fp16."""
import gc
import math

import numpy as np
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, make
from tests.test_gpu_shared import make_shared, vectors

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


# ---- accumulated weights -----------------------------------------------------------------------------------------------

def logits_of(specs, q, b, n, new, token, layer, h, window, sinks, gone=()):
    group = q.shape[1] // specs["kv_data"].shape[3]
    (xk, zk), _ = vectors(specs, specs["kv_indptr"], b, n, layer, h)
    for s, p in gone:
        if s == b:
            xk[p], zk[p] = 0, 0
    qs = q[token:token + new, h * group:(h + 1) * group].reshape(-1, 128).double()
    place, j = torch.arange(n - new, n, device=DEV)[:, None].repeat(1, group).reshape(-1, 1), torch.arange(n, device=DEV)[None]
    sees = (j <= place) & ((place - j < window) | (j < sinks) if window else True)
    for s, p in gone:
        if s == b:
            sees[:, p] = False
    logits = (qs @ xk.T - qs.sum(1, keepdim=True) * zk.T) / math.sqrt(128)
    terms = (qs.abs() @ xk.abs().T + qs.abs().sum(1, keepdim=True) * zk.abs().T) / math.sqrt(128)
    return logits, terms, sees


def logarithms(specs, q, lens, news, layer=1, window=0, sinks=0, gone=()):
    lse = torch.full(q.shape[:2], -math.inf, device=DEV)
    heads = specs["kv_data"].shape[3]
    group, token = q.shape[1] // heads, 0
    for b, (n, new) in enumerate(zip(lens, news)):
        if n and new:
            for h in range(heads):
                logits, _, sees = logits_of(specs, q, b, n, new, token, layer, h, window, sinks, gone)
                lse[token:token + new, h * group:(h + 1) * group] = torch.logsumexp(torch.where(sees, logits, -math.inf), 1).reshape(new, group).float()
        token += new
    return lse


def definition(specs, q, lse, start, lens, news, layer=1, window=0, sinks=0, gone=()):
    heads, capacity = specs["kv_data"].shape[3], start.shape[2]
    group, token = q.shape[1] // heads, 0
    want, tol = start.double(), 2.0 ** -23 * start.double().abs()
    for b, (n, new) in enumerate(zip(lens, news)):
        if n and new:
            for h in range(heads):
                logits, terms, sees = logits_of(specs, q, b, n, new, token, layer, h, window, sinks, gone)
                of = lse[token:token + new, h * group:(h + 1) * group].reshape(-1, 1).double()
                p = torch.where(sees & (of > -math.inf), torch.exp(logits - of), 0.0)
                off = torch.where(p > 0, p * (140 * 2.0 ** -24 * terms + 2.0 ** -21 * (1 + logits.abs() + of.abs())), 0.0)
                m = min(n, capacity)
                want[b, h, :m] += p.sum(0)[:m]
                tol[b, h, :m] += (off.sum(0) + 2.0 ** -16 * p.sum(0))[:m] + 2.0 ** -23 * want[b, h, :m].abs() + 1e-37
        token += new
    return want, tol


def check(specs, q, starts, lens, news, layer=1, window=0, sinks=0, gone=(), capacity=None, step=False, lse=None, hints=(False, True), **kw):
    heads, batch = specs["kv_data"].shape[3], len(lens)
    capacity = max(1, *lens) + 5 if capacity is None else capacity
    start = torch.rand(batch, heads, capacity, generator=torch.Generator().manual_seed(len(lens))).to(DEV)
    lse = logarithms(specs, kw.get("q_in", q), lens, news, layer, window, sinks, gone) if lse is None else lse
    want, tol = definition(specs, kw.pop("q_in", q), lse, start, lens, news, layer, window, sinks, gone)
    call = kv.accumulate_weights_f16 if specs["kv_data"].dtype == torch.float16 else kv.accumulate_weights_i4
    for hint in hints:
        behind = torch.full((batch * heads * capacity + 64,), 7.0, device=DEV)
        got = behind[:batch * heads * capacity].view(batch, heads, capacity).copy_(start)
        given = {"max_new_len": max(news), "max_seq_len": max(lens)} if hint else {}
        assert call(got, q, lse, **specs, layer_idx=layer, seqlen_indptr=None if step else starts, window=window, sinks=sinks, **given, **kw) is None
        off = (got.double() - want).abs()
        assert bool((off <= tol).all()), f"hint {hint}: {float((off / tol.clamp(min=1e-30)).max())} of what is allowed, at {(off - tol).argmax().item()}"
        assert bool((behind[batch * heads * capacity:] == 7).all())
    return got


SHAPES = [                                                  # page size, tokens held, new ones
    (16, [1], [1]), (16, [5], [5]), (16, [17, 64, 1], [1, 64, 1]), (16, [700, 33, 129], [3, 33, 100]), (64, [64, 1000, 63], [64, 7, 2]), (128, [300, 128], [257, 1]),
    (5, [11, 1, 64], [3, 1, 40]), (7, [200, 20], [150, 20]), (2048, [2048, 31], [9, 31]), (1, [40], [12]), (16, [40, 0, 9, 30], [4, 0, 0, 30]), (16, [3, 0, 20], [7, 4, 5]),
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,group", [(4, 1), (2, 8), (3, 3), (1, 5)])
@pytest.mark.parametrize("page_size,lens,news", SHAPES)
def test_weights_of_all_lengths(page_size, lens, news, heads, group, f16):
    specs, q, starts = make(page_size * 5 + len(lens), page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (33, 0), (100, 40), (64, 1000), (5000, 3)])
@pytest.mark.parametrize("page_size,lens,news,heads,group", [(16, [700, 33, 129], [90, 33, 1], 2, 4), (5, [64, 300], [64, 20], 3, 1), (64, [1500], [200], 1, 8)])
def test_weights_in_windows(page_size, lens, news, heads, group, window, sinks, f16):
    specs, q, starts = make(window + sinks, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (128, 4)])
@pytest.mark.parametrize("page_size,lens,heads,group", [(16, [1, 500, 4001], 4, 1), (32, [3000] * 2, 2, 8), (7, [90, 1000], 5, 2), (128, [9000], 1, 16), (16, [900], 1, 40)])
def test_weights_of_one_token_per_sequence(page_size, lens, heads, group, window, sinks, f16):
    news = [1] * len(lens)
    specs, q, starts = make(page_size + window, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks, step=True)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,lens,news,heads,group,window,sinks", [
    (16, [600], [600], 2, 1, 0, 0), (16, [1500, 300, 2], [257, 300, 2], 1, 4, 0, 0), (64, [2000], [700], 2, 3, 0, 0), (5, [900], [400], 1, 2, 0, 0),
    (7, [400, 90], [300, 0], 1, 1, 100, 4), (16, [3000], [513], 1, 5, 500, 70), (128, [1000, 1000], [40, 999], 1, 8, 64, 1), (16, [70, 5], [200, 9], 2, 2, 0, 0),
    (16, [4100], [2100], 1, 8, 0, 0)])
def test_weights_of_many_rows(page_size, lens, news, heads, group, window, sinks, f16):
    specs, q, starts = make(page_size + heads, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("lens,news,group,window,sinks", [([1500], [1400], 8, 0, 0), ([300, 1100], [300, 1000], 6, 0, 0), ([2600], [1200], 8, 300, 20), ([700, 0, 90], [600, 0, 90], 20, 0, 0)])
def test_weights_of_rows_in_parts(lens, news, group, window, sinks, f16):
    """Few blocks of positions and many rows, which several workgroups share; hints that are too small leave blocks to one workgroup, too large ones leave workgroups without a block."""
    specs, q, starts = make(sum(lens), 16, lens, news, 1, group, f16)
    lse = logarithms(specs, q, lens, news, window=window, sinks=sinks)
    check(specs, q, starts, lens, news, window=window, sinks=sinks, lse=lse)
    start = torch.rand(len(lens), 1, max(lens), device=DEV)
    want, tol = definition(specs, q, lse, start, lens, news, window=window, sinks=sinks)
    call = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4
    for new, length in ((0, 1), (max(news), 200), (0, 40000), (1, 0), (100000, 1 << 40)):
        got = start.clone()
        call(got, q, lse, **specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=length, window=window, sinks=sinks,
             workspace=torch.full((1 << 26,), 255, dtype=torch.uint8, device=DEV))
        assert bool(((got.double() - want).abs() <= tol).all()), (new, length)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[40, 90], [1, 1], [300, 20]])
def test_weights_of_large_logits(f16, news):
    lens = [600, 90]
    specs, q, starts = make(5, 16, lens, news, 2, 2, f16, spread=12.0)
    check(specs, q, starts, lens, news)
    if not f16:
        specs["kv_param"][:, :, 0, :, ::3, 0] = 0
        specs["kv_param"][:, :, 0, :, 1::3, 0] *= -1
        check(specs, q, starts, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[20, 30], [1, 1], [50, 400]])
@pytest.mark.parametrize("page_size", [16, 6])
def test_weights_where_pages_are_missing_and_capacity_ends(page_size, news, f16):
    lens = [50, 490]
    specs, q, starts = make(9, page_size, lens, news, 2, 2, f16)
    at = int(specs["kv_indptr"][1])
    specs["kv_indices"][1], specs["kv_indices"][at + 2] = specs["kv_data"].shape[0], -5
    clean = specs["kv_indices"].clone()
    clean[1], clean[at + 2] = 0, 0
    gone = [(0, p) for p in range(page_size, 2 * page_size)] + [(1, p) for p in range(2 * page_size, 3 * page_size)]
    # (the definition reads page 0 there and takes it out; a finite one)
    for name in ("kv_data", "kv_param"):
        if specs[name].dtype == torch.float16:
            specs[name].nan_to_num_(nan=0.5)
    lse = logarithms({**specs, "kv_indices": clean}, q, lens, news, gone=gone)
    heads = 2
    for capacity in (495, 300, 17):
        start = torch.rand(2, heads, capacity, device=DEV)
        want, tol = definition({**specs, "kv_indices": clean}, q, lse, start, lens, news, gone=gone)
        got = torch.cat([start.flatten(), torch.full((64,), 7.0, device=DEV)])
        call = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4
        call(got[:start.numel()].view(start.shape), q, lse, **specs, layer_idx=1, seqlen_indptr=starts)
        assert bool(((got[:start.numel()].view(start.shape).double() - want).abs() <= tol).all()) and bool((got[start.numel():] == 7).all())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[3, 9], [1, 1], [70, 200]])
def test_nans_and_infinities_reach_only_what_sees_them(news, f16):
    """A key that is no number reaches its position, a query row the positions that it sees, a logarithm of -inf nothing; all other sums are the same bits."""
    lens = [90, 300]
    specs, q, starts = make(10, 16, lens, news, 2, 2, f16)
    lse = logarithms(specs, q, lens, news)
    call = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4

    def run(specs, q, lse):
        got = torch.zeros(2, 2, 310, device=DEV)
        call(got, q, lse, **specs, layer_idx=1, seqlen_indptr=starts)
        return got

    clean = run(specs, q, lse)
    page = int(specs["kv_indices"][1])
    bad = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
    if f16:
        bad["kv_data"][page, 1, 0, :, 4, 7] = float("nan")
    else:
        bad["kv_param"][page, 1, 0, :, 4, 0] = float("nan")
    got = run(bad, q, lse)
    assert bool(torch.isnan(got[0, :, 20]).all())
    got[0, :, 20] = clean[0, :, 20]
    assert torch.equal(got, clean)
    row = q.clone()
    row[news[0]:news[0] + 1, :2] = float("nan")             # the second sequence's first row, of the first key head
    got = run(specs, row, lse)
    first = lens[1] - news[1]
    assert bool(torch.isnan(got[1, 0, :first + 1]).all())
    got[1, 0, :first + 1] = clean[1, 0, :first + 1]
    assert torch.equal(got, clean)
    none = lse.clone()
    none[0] = -math.inf
    want, tol = definition(specs, q, none, torch.zeros_like(clean), lens, news)
    assert bool(((run(specs, q, none).double() - want).abs() <= tol).all())
    never = lse.clone()
    never[0] = math.inf
    assert torch.equal(run(specs, q, never), run(specs, q, none))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[33, 30], [1, 1], [300, 30]])
def test_weights_of_strided_queries_and_the_transform(news, f16):
    lens = [370, 30]
    specs, q, starts = make(11, 16, lens, news, 2, 4, f16, fused=512)
    assert q.stride(0) == 8 * 128 + 512
    check(specs, q, starts, lens, news)
    qh = kv.matmul_had_cuda(q.contiguous(), torch.float16)
    lse = logarithms(specs, qh, lens, news)
    inside, apart = torch.zeros(2, 2, 370, device=DEV), torch.zeros(2, 2, 370, device=DEV)
    call = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4
    call(inside, q, lse, **specs, layer_idx=1, seqlen_indptr=starts, q_hadamard=True)
    call(apart, qh, lse, **specs, layer_idx=1, seqlen_indptr=starts)
    # (an element of the transform may be rounded to the other side: 2^-11 of it)
    assert float((inside - apart).double().norm() / apart.double().norm()) < 2.0 ** -9


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("batch,most,group", [(70, 70, 8), (130, 3, 8)])
def test_weights_of_many_sequences(batch, most, group, f16):
    news = [(7 * b) % (most + 1) for b in range(batch)]
    lens = [n + (13 * b) % 90 for b, n in enumerate(news)]
    specs, q, starts = make(batch, 16, lens, news, 2, group, f16)
    check(specs, q, starts, lens, news)


@pytest.mark.parametrize("new", [1, 60])
def test_weights_captured_and_the_same_bits(new):
    lens, news = [3000, 1500], [new, new]
    specs, q, starts = make(14, 16, lens, news, 2, 4)
    lse = logarithms(specs, q, lens, news)
    args = dict(**specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=3000)
    eager, sums = torch.zeros(2, 2, 3000, device=DEV), torch.zeros(2, 2, 3000, device=DEV)
    kv.accumulate_weights_i4(eager, q, lse, **args)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.accumulate_weights_i4(sums, q, lse, **args)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    kv.accumulate_weights_i4(eager, q, lse, **args)
    kv.accumulate_weights_i4(eager, q, lse, **args)
    assert torch.equal(sums, eager)


# ---- which stay --------------------------------------------------------------------------------------------------------

def stays(weights, lengths, keep, sinks, recent):
    batch, heads, capacity = weights.shape
    kept = np.full((batch, heads, keep), -1, dtype=np.int32)
    lengths = np.clip(lengths, 0, capacity)
    for b in range(batch):
        n = int(lengths[b])
        for h in range(heads):
            if n <= keep:
                kept[b, h, :n] = np.arange(n)
                continue
            w = weights[b, h, sinks:n - recent].astype(np.float64)
            rank = np.where(np.isnan(w), -np.inf, w)
            # (NaN behind an infinity below all numbers too)
            order = sorted(range(len(w)), key=lambda i: (-rank[i], bool(np.isnan(w[i])), i)) if np.isnan(w).any() else np.argsort(-rank, kind="stable")
            between = np.sort(np.asarray(order[:keep - sinks - recent], dtype=np.int64)) + sinks
            kept[b, h] = np.concatenate([np.arange(sinks), between, np.arange(n - recent, n)])
    return kept, np.minimum(lengths, keep).astype(np.int32)


def check_heavy(weights, lengths, keep, sinks=0, recent=0):
    want, left = stays(weights.numpy(), np.asarray(lengths), keep, sinks, recent)
    kept, new_lengths = kv.heavy_positions(weights.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), keep, sinks=sinks, recent=recent)
    assert kept.dtype == new_lengths.dtype == torch.int32
    np.testing.assert_array_equal(new_lengths.cpu().numpy(), left)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)


@pytest.mark.parametrize("lengths,capacity,keep,sinks,recent", [
    ([1], 1, 1, 0, 0), ([5, 0, 3], 8, 3, 1, 1), ([100, 64, 65, 63], 100, 64, 4, 16), ([700, 3, 701], 701, 300, 0, 0), ([3000] * 3, 4000, 1024, 4, 256), ([2000, -7, 9000], 2500, 999, 100, 0),
    ([40001], 40001, 5000, 4, 1000), ([1025], 1025, 1024, 0, 0), ([1025], 1025, 1, 0, 0), ([500], 500, 10, 10, 0), ([500], 500, 10, 0, 10), ([500], 500, 10, 4, 6), ([77], 77, 0, 0, 0),
    ([300], 300, 5000, 4, 100), ([70000], 70000, 33000, 0, 7)])
def test_positions_that_stay(lengths, capacity, keep, sinks, recent):
    g = torch.Generator().manual_seed(capacity + keep)
    weights = torch.exp(2 * torch.randn(len(lengths), 3, capacity, generator=g) - 3)
    weights[torch.rand(weights.shape, generator=g) < 0.05] = 0
    check_heavy(weights, lengths, keep, sinks, recent)


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 0), (100, 4, 20), (511, 0, 0), (700, 1, 100)])
@pytest.mark.parametrize("kind", ["equal", "few", "steps", "signs", "bits", "odd", "one bit"])
def test_equal_negative_and_odd_sums(kind, keep, sinks, recent):
    """Ties at every digit, negative sums, both zeros, infinities and NaN."""
    g = torch.Generator().manual_seed(keep)
    n = 1500
    weights = {"equal": torch.full((2, 2, n), 0.25), "few": torch.randint(0, 3, (2, 2, n), generator=g).float(), "steps": torch.randint(0, 40, (2, 2, n), generator=g) / 8.0,
               "signs": torch.randn(2, 2, n, generator=g).round(decimals=1), "bits": torch.randint(-(2 ** 31), 2 ** 31 - 1, (2, 2, n), generator=g, dtype=torch.int64).to(torch.int32).view(torch.float32),
               "odd": torch.randn(2, 2, n, generator=g), "one bit": (torch.randint(0, 2, (2, 2, n), generator=g, dtype=torch.int32) + 0x3F800000).view(torch.float32)}[kind].clone()
    if kind == "odd":
        weights[torch.rand(weights.shape, generator=g) < 0.2] = math.inf
        weights[torch.rand(weights.shape, generator=g) < 0.2] = -math.inf
        weights[torch.rand(weights.shape, generator=g) < 0.3] = math.nan
        weights[0, 0] = math.nan
    if kind == "signs":
        weights[weights == 0] = -0.0
        weights[..., ::7] = 0.0
    check_heavy(weights, [n, n - 1], keep, sinks, recent)


# ---- their move --------------------------------------------------------------------------------------------------------

def bits(t):
    return t.view(torch.int16) if t.dtype == torch.float16 else t


def check_keep(specs, lens, kept, layer, weights=None):
    """Against a move on the host, position by position; everything else keeps its bits."""
    heads, page = specs["kv_data"].shape[3:5]
    want = {name: bits(specs[name]).clone() for name in ("kv_data", "kv_param")}
    want_w = None if weights is None else weights.clone()
    bounds, pages = specs["kv_indptr"].tolist(), specs["kv_indices"].long()
    total = specs["kv_data"].shape[0]
    for b, n in enumerate(lens):
        table = pages[bounds[b]:bounds[b + 1]]
        for h in range(heads):
            source = kept[b, h].long()
            to = torch.arange(source.numel(), device=DEV)
            good = (source >= 0) & (source < n) & (to < n)
            source, to = source[good], to[good]
            real = (table[source // page] >= 0) & (table[source // page] < total) & (table[to // page] >= 0) & (table[to // page] < total)
            s, t = source[real], to[real]
            for name in want:
                rows = bits(specs[name])[table[s // page], layer, :, h, s % page]
                want[name][table[t // page], layer, :, h, t % page] = rows
            if weights is not None:
                have = min(n, weights.shape[2])
                inside = (source < have) & (to < have)
                want_w[b, h, :have] = 0
                want_w[b, h, to[inside]] = weights[b, h, source[inside]]
    got_w = None if weights is None else weights.clone()
    call = kv.keep_positions_f16 if specs["kv_data"].dtype == torch.float16 else kv.keep_positions_i4
    assert call(kept, **specs, layer_idx=layer, weights=got_w) is None
    for name in want:
        assert torch.equal(bits(specs[name]), want[name]), name
    assert weights is None or torch.equal(got_w, want_w)


def random_lists(seed, lens, heads, keep):
    g = torch.Generator().manual_seed(seed)
    kept = torch.full((len(lens), heads, keep), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for h in range(heads):
            some = torch.randperm(n, generator=g)[:keep].sort().values
            kept[b, h, :some.numel()] = some.int()
    return kept.to(DEV)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,lens,heads,keep", [
    (16, [1], 1, 1), (16, [40, 17, 300], 3, 16), (16, [2000, 5], 2, 1030), (64, [1000], 4, 999), (7, [100, 33], 2, 50), (1, [60], 2, 20), (128, [3000, 0, 200], 2, 700),
    (5, [4000], 1, 2500), (16, [90], 2, 200), (16, [50], 2, 0)])
def test_moves(page_size, lens, heads, keep, f16):
    specs, _, _ = make(page_size + keep, page_size, lens, [0] * len(lens), heads, 1, f16)
    kept = random_lists(keep, lens, heads, keep)
    weights = torch.rand(len(lens), heads, max(lens) + 3, device=DEV)
    check_keep(specs, lens, kept, 1, weights)
    check_keep(specs, lens, kept, 0)


@pytest.mark.parametrize("f16", [False, True])
def test_moves_of_edges(f16):
    """Nothing moves; only the first, or the last go; weights that end before the sequence; entries and page numbers that are none."""
    lens, heads = [600, 600, 600, 600], 2
    specs, _, _ = make(3, 16, lens, [0] * 4, heads, 1, f16)
    at = torch.arange(599, dtype=torch.int32)
    kept = torch.stack([at, at + 1, torch.cat([at[:300], at[300:] + 1]), torch.cat([at[:1], at[1:] + 1])])[:, None].repeat(1, heads, 1).contiguous().to(DEV)
    check_keep(specs, lens, kept, 1, torch.rand(4, heads, 350, device=DEV))
    specs["kv_indices"][3], specs["kv_indices"][5] = -1, specs["kv_data"].shape[0]
    kept = random_lists(4, lens, heads, 200)
    kept[1, :, 150:] = 600 + torch.arange(50, dtype=torch.int32, device=DEV)
    kept[2, :, 100:] = -1
    check_keep(specs, lens, kept, 0, torch.rand(4, heads, 700, device=DEV))


# ---- together ----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("prefix_len", [0, 200])
def test_prompt_steps_eviction_and_on(prefix_len, f16):
    """A prompt, steps and drafted tokens of a ragged batch, with or without a shared prefix: attention with its logarithms, sums of weights, then half of every
    key head's positions go, new tables, and further tokens attend to what stayed.  After the eviction attention is the definition's over the
    vectors that the lists name."""
    page, heads, group, layers = 16, 2, 4, 2
    most, batch = [300, 120, 77], 3
    room = [n + 60 for n in most]
    g = torch.Generator().manual_seed(prefix_len + f16)
    specs, prefix, _, _ = make_shared(1, page, [prefix_len or 1], None, room, [0] * batch, heads, group, f16)
    table = torch.zeros(batch, 32, dtype=torch.int32, device=DEV)
    bounds = specs["kv_indptr"].tolist()
    for b in range(batch):
        table[b, :bounds[b + 1] - bounds[b]] = specs["kv_indices"][bounds[b]:bounds[b + 1]]
    pool = {name: specs[name] for name in ("kv_data", "kv_param")}
    for name in pool:
        if pool[name].dtype == torch.float16:
            pool[name].nan_to_num_(nan=0.25)
    shared = dict(prefix) if prefix_len else None
    accumulate = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4
    move = kv.keep_positions_f16 if f16 else kv.keep_positions_i4
    weights = torch.zeros(layers, batch, heads, 400, device=DEV)
    lengths = torch.zeros(batch, dtype=torch.int32, device=DEV)

    def turn(news, lengths):
        """The new tokens' vectors are what lies in the pages; returns the outputs of both layers."""
        lengths = lengths + torch.tensor(news, dtype=torch.int32, device=DEV)
        t = kv.build_page_tables(lengths, page, 32, block_table=table, new_lengths=torch.tensor(news, dtype=torch.int32, device=DEV), tokens=sum(news))
        tables = {name: t[name] for name in ("kv_indptr", "kv_indices", "last_page_offset")}
        outs = []
        for layer in range(layers):
            q = torch.randn(sum(news), heads * group, 128, generator=g).half().to(DEV)
            o, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
            if shared:
                (kv.batch_shared_f16 if f16 else kv.batch_shared_i4)(o, q, **pool, **tables, layer_idx=layer, **shared, seqlen_indptr=t["seqlen_indptr"], lse=lse)
            else:
                (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **pool, **tables, layer_idx=layer, seqlen_indptr=t["seqlen_indptr"], lse=lse)
            accumulate(weights[layer], q, lse, **pool, **tables, layer_idx=layer, seqlen_indptr=t["seqlen_indptr"])
            outs.append((q, o))
        return lengths, tables, outs

    from tests.test_gpu_chunk import definition as attention
    lengths, tables, _ = turn(most, lengths)
    for news in ([1, 1, 1], [5, 1, 3]):
        lengths, tables, _ = turn(news, lengths)
    held = lengths.tolist()
    # every row's weights add up to one (less what the prefix has)
    rows = [sum(n) for n in zip(most, [1, 1, 1], [5, 1, 3])]
    for b in range(batch):
        total = weights[:, b].double().sum(-1)
        assert bool((total <= rows[b] * group * (1 + 2.0 ** -10)).all())
        assert prefix_len or bool((total >= rows[b] * group * (1 - 2.0 ** -10)).all())
        assert bool((weights[:, b, :, held[b]:] == 0).all())
    keep = 100
    before = {name: pool[name].clone() for name in pool}
    lists = []
    for layer in range(layers):
        kept, new_lengths = kv.heavy_positions(weights[layer], lengths, keep, sinks=4, recent=20)
        np.testing.assert_array_equal(kept.cpu().numpy(), stays(weights[layer].cpu().numpy(), np.asarray(held), keep, 4, 20)[0])
        sums = weights[layer].clone()
        move(kept, **pool, **tables, layer_idx=layer, weights=weights[layer])
        for b in range(batch):
            n = int(new_lengths[b])
            assert torch.equal(weights[layer, b, :, :n], torch.gather(sums[b], 1, kept[b, :, :n].long())) and bool((weights[layer, b, :, n:] == 0).all())
        lists.append(kept)
    lengths = new_lengths
    assert lengths.tolist() == [min(n, keep) for n in held]
    # the vectors in front are the lists'
    bounds, at = tables["kv_indptr"].tolist(), tables["kv_indices"].long()
    for layer, kept in enumerate(lists):
        for b in range(batch):
            n, mine = int(lengths[b]), at[bounds[b]:bounds[b + 1]]
            for h in range(heads):
                s, t = kept[b, h, :n].long(), torch.arange(n, device=DEV)
                for name in pool:
                    assert torch.equal(bits(pool[name])[mine[t // page], layer, :, h, t % page], bits(before[name])[mine[s // page], layer, :, h, s % page])
    news = [2, 1, 4]
    lengths, tables, outs = turn(news, lengths)
    for layer, (q, o) in enumerate(outs):
        if shared:
            from tests.test_gpu_shared import definition as joined
            (want, tol), _ = joined({**pool, **tables, "kv_indices": torch.cat([tables["kv_indices"], prefix["prefix_indices"]])},
                                    {**prefix, "prefix_indptr": prefix["prefix_indptr"] + tables["kv_indices"].numel()}, q, [prefix_len], None, lengths.tolist(), news, layer)
        else:
            want, tol = attention({**pool, **tables}, q, lengths.tolist(), news, layer)
        assert bool(((o.double() - want).abs() <= tol).all())


def test_refusals():
    lens, news = [20, 5], [3, 2]
    specs, q, starts = make(17, 16, lens, news, 2, 2)
    lse, w = torch.zeros(q.shape[:2], device=DEV), torch.zeros(2, 2, 20, device=DEV)
    run = lambda **kw: kv.accumulate_weights_i4(**{"weights": w, "q": q, "lse": lse, **specs, "layer_idx": 1, "seqlen_indptr": starts, **kw})
    run()
    for match, kw in (("weights", {"weights": w.double()}), ("weights", {"weights": w[:1]}), ("weights", {"weights": w[:, :, ::2]}), ("weights", {"weights": w[0]}), ("lse", {"lse": lse.half()}),
                      ("lse", {"lse": lse[:, :3]}), ("lse", {"lse": lse.cpu()}), ("fp16", {"q": q.float()}), ("contiguous heads", {"q": q.transpose(0, 1).contiguous().transpose(0, 1)}),
                      ("multiple of the cache", {"q": q[:, :3].contiguous(), "lse": lse[:, :3].contiguous()}), ("one token per sequence", {"seqlen_indptr": None}), ("negative", {"window": -1}),
                      ("negative", {"max_new_len": -1}), ("layer_idx", {"layer_idx": -1}), ("uint8", {"kv_data": specs["kv_data"].half()}), ("batch_size", {"kv_indptr": specs["kv_indptr"][:2]})):
        with pytest.raises(RuntimeError, match=match):
            run(**kw)
    with pytest.raises(RuntimeError, match="fp16"):
        kv.accumulate_weights_f16(w, q, lse, **specs, layer_idx=1, seqlen_indptr=starts)
    run(q=q[:0], lse=lse[:0], seqlen_indptr=starts * 0)
    n = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for match, args, kw in (("weights", (w.half(), n, 4), {}), ("weights", (w.cpu(), n.cpu(), 4), {}), ("lengths", (w, n.long(), 4), {}), ("lengths", (w, n[:1], 4), {}), ("lengths", (w, n.cpu(), 4), {}),
                            ("sinks", (w, n, 4), {"sinks": 3, "recent": 2}), ("sinks", (w, n, 4), {"sinks": -1}), ("sinks", (w, n, -1), {}), ("sinks", (w, n, 4), {"recent": -1})):
        with pytest.raises(RuntimeError, match=match):
            kv.heavy_positions(*args, **kw)
    kept, _ = kv.heavy_positions(w, n, 4)
    move = lambda **kw: kv.keep_positions_i4(**{"kept": kept, **specs, "layer_idx": 1, "weights": w, **kw})
    move()
    for match, kw in (("kept", {"kept": kept.long()}), ("kept", {"kept": kept[:1]}), ("kept", {"kept": kept[0]}), ("kept", {"kept": kept[:, :, ::2]}), ("weights", {"weights": w[:, :1]}),
                      ("weights", {"weights": w.cpu()}), ("layer_idx", {"layer_idx": 2}), ("batch_size", {"kv_indptr": specs["kv_indptr"][:2]})):
        with pytest.raises(RuntimeError, match=match):
            move(**kw)
    empty, left = kv.heavy_positions(w[:0], n[:0], 4)
    assert tuple(empty.shape) == (0, 2, 4) and tuple(left.shape) == (0,)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[3, 9], [1, 1], [2, 8], [70, 200], [33, 400]])
def test_rows_that_give_nothing_may_hold_anything(news, f16):
    """A row whose logarithm is -inf gives nothing, whatever its queries are (rows that a caller leaves out): the bits of a call with zeros there."""
    lens = [90, 500]
    specs, q, starts = make(15, 16, lens, news, 2, 8, f16)
    lse = logarithms(specs, q, lens, news)
    out = [0, news[0], sum(news) - 1]
    call = kv.accumulate_weights_f16 if f16 else kv.accumulate_weights_i4
    sums = []
    for value in (0.0, math.nan, math.inf):
        row, of = q.clone(), lse.clone()
        row[out, 3:11], of[out, 3:11] = value, -math.inf
        row[out, 3:11, ::2] *= -1
        got = torch.zeros(2, 2, 510, device=DEV)
        call(got, row, of, **specs, layer_idx=1, seqlen_indptr=starts)
        sums.append(got)
    assert bool((sums[0] != 0).any()) and torch.equal(sums[1], sums[0]) and torch.equal(sums[2], sums[0])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [1, 40])
def test_a_turn_with_eviction_captured_and_replayed(new, f16):
    """Attention, its weights, which stay and their move in one graph, replayed with eager work between: the bits of as many eager turns.  The lengths and page tables are
    those from before every turn, so each moves what the last has left."""
    lens, news = [700, 300], [new, new]
    specs, q, starts = make(16, 16, lens, news, 2, 4, f16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    suffix = "_f16" if f16 else "_i4"
    chunk, accumulate, move = (getattr(kv, name + suffix) for name in ("batch_chunk", "accumulate_weights", "keep_positions"))

    def state():
        return {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}, torch.zeros(2, 2, 700, device=DEV), torch.zeros_like(q), torch.zeros(q.shape[:2], device=DEV)

    def turn(specs, sums, o, lse):
        how = dict(**specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=700)
        chunk(o, q, **how, lse=lse)
        accumulate(sums, q, lse, **how)
        kept, _ = kv.heavy_positions(sums, lengths, 200, sinks=4, recent=50)
        move(kept, **specs, layer_idx=1, weights=sums)

    eager, captured, warm = state(), state(), state()
    turn(*warm)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turn(*captured)
    for _ in range(4):
        graph.replay()
        turn(*eager)
        torch.cuda.synchronize()
        for have, want in zip((captured[0]["kv_data"], captured[0]["kv_param"], *captured[1:]), (eager[0]["kv_data"], eager[0]["kv_param"], *eager[1:])):
            assert torch.equal(bits(have), bits(want))


def test_evictions_on_two_streams_at_once():
    """Two caches' turns under way together, each on a stream of its own: the bits of one after the other."""
    lens, news = [2000, 900], [30, 5]
    cases = []
    for seed in (17, 18):
        specs, q, starts = make(seed, 16, lens, news, 2, 4)
        cases.append((specs, q, starts, logarithms(specs, q, lens, news)))
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def turn(specs, q, starts, lse):
        specs = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
        sums = torch.zeros(2, 2, 2000, device=DEV)
        kv.accumulate_weights_i4(sums, q, lse, **specs, layer_idx=1, seqlen_indptr=starts)
        kept, left = kv.heavy_positions(sums, lengths, 500, sinks=4, recent=50)
        kv.keep_positions_i4(kept, **specs, layer_idx=1, weights=sums)
        return specs["kv_data"], specs["kv_param"], sums, kept, left

    alone = [turn(*case) for case in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        together = []
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                together.append(turn(*case))
        torch.cuda.synchronize()
        for got, want in zip(together, alone):
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))

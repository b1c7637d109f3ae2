"""Attention of new tokens over the paged cache (batch_chunk_i4, batch_chunk_f16) against its definition in 64 bits.

How far a result may be off is added up for every element.  With weights w_j (they add up to one), values v_j, x_j = scale_j code (and
zero_j, subtracted from it) on int4 pages, and half a step of fp16 being u = 2^-11:
  u |o|                                   the output's rounding (2^-25 where it is subnormal)
  u (sum w_j |v_j| + |o|)                 a weight is rounded to fp16 once and counts as rounded in all sums: w_j (1 + d_j), |d_j| <= u, changes
                                          sum w v / sum w by sum w_j d_j (v_j - o), at most u sum w_j |v_j - o|
  sum min(w_j, 2^-25) (|v_j| + |o|)       the same for weights below fp16's normal range; sums are at least one in units of the largest weight
  L sum w_j (|x_j| + |zero_j|)            with L twice the largest error of a logit -- 140 steps of 2^-24 of its terms' absolute sum, and for queries
                                          below 2^-10 a step of 2^-21 of a sixteenth of them --, plus that of exp2's argument and of sums over the
                                          positions, all in fp32."""
import gc
import math

import numpy as np
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


def make(seed, page_size, lens, news, heads, group, f16=False, layers=2, spare=3, fused=0, spread=1.0):
    """A cache of random vectors, its page tables, and queries; pages scattered over the pool, the unused ones full of NaN."""
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // page_size) for n in lens]
    total = sum(per) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    shape = (total, layers, 2, heads, page_size)
    if f16:
        data = torch.randn(*shape, 128, generator=g).half()
        param = torch.full((*shape, 2), float("nan"), dtype=torch.float16)              # not read
    else:
        data = torch.randint(0, 256, (*shape, 64), generator=g, dtype=torch.uint8)
        scale = 0.05 + 0.5 * torch.rand(*shape, 1, generator=g)
        param = torch.cat([scale, scale * 7.5 + 0.3 * torch.randn(*shape, 1, generator=g)], -1).half()
    # what no sequence holds may be anything
    used = torch.zeros(total, page_size, dtype=torch.bool)
    at = 0
    for n, p in zip(lens, per):
        for i in range(p):
            used[order[at + i], :min(page_size, n - i * page_size)] = True
        at += p
    hole = ~used[:, None, None, None, :].expand(shape)
    (data if f16 else param)[hole] = float("nan")
    tokens = sum(news)
    q = (torch.randn(tokens, heads * group * 128 + fused, generator=g) * spread).half()
    start = lambda v: torch.tensor(np.concatenate([[0], np.cumsum(v)]).astype(np.int32))
    last = [n - (p - 1) * page_size if p else 0 for n, p in zip(lens, per)]
    specs = {"kv_data": data, "kv_param": param, "kv_indptr": start(per), "kv_indices": order, "last_page_offset": torch.tensor(last, dtype=torch.int32)}
    specs = {k: v.to(DEV) for k, v in specs.items()}
    return specs, q.to(DEV)[:, :heads * group * 128].view(tokens, heads * group, 128), start(news).to(DEV)


def definition(specs, q, lens, news, layer, window=0, sinks=0, gone=()):
    """(result, how far off) in 64 bits; `gone`: (sequence, position) pairs that are not there."""
    data, param, f16 = specs["kv_data"], specs["kv_param"], specs["kv_data"].dtype == torch.float16
    heads, page_size = data.shape[3], data.shape[4]
    group = q.shape[1] // heads
    bounds, pages = specs["kv_indptr"].tolist(), specs["kv_indices"].long()
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    token = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        if new and n:
            held = pages[bounds[b]:bounds[b + 1]].clamp(0, data.shape[0] - 1)
            place = torch.arange(n - new, n, device=DEV)[:, None].repeat(1, group).reshape(-1, 1)
            j = torch.arange(n, device=DEV)[None]
            sees = j <= place
            if window:
                sees &= (place - j < window) | (j < sinks)
            for s, p in gone:
                if s == b:
                    sees[:, p] = False
            for h in range(heads):
                x, z = [], []
                for side in (0, 1):
                    rows = data[held, layer, side, h].reshape(-1, data.shape[-1])[:n]
                    if f16:
                        x.append(rows.double()), z.append(torch.zeros(n, 1, dtype=torch.float64, device=DEV))
                    else:
                        pr = param[held, layer, side, h].reshape(-1, 2)[:n].double()
                        codes = torch.stack([rows & 15, rows >> 4], -1).reshape(n, 128).double()
                        x.append(pr[:, :1] * codes), z.append(pr[:, 1:])
                for s, p in gone:                           # (not to be read, whatever lies where its page number leads here)
                    if s == b:
                        for v in (*x, *z):
                            v[p] = 0
                qs = q[token:token + new, h * group:(h + 1) * group].reshape(-1, 128).double()
                logits = (qs @ x[0].T - qs.sum(1, keepdim=True) * z[0].T) / math.sqrt(128)
                terms = (qs.abs() @ x[0].abs().T + qs.abs().sum(1, keepdim=True) * z[0].abs().T) / math.sqrt(128)
                masked = torch.where(sees, logits, -math.inf)
                w = torch.exp(masked - masked.amax(1, keepdim=True).clamp(min=-1e300))
                w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
                w = torch.where(sees, w, 0.0)
                o = w @ (x[1] - z[1])
                size = w @ (x[1].abs() + z[1].abs())
                small = 2.0 ** -21 * x[0].abs().sum(1)[None] / math.sqrt(128)
                far = 2 * torch.where(sees, 140 * 2.0 ** -24 * terms + small, 0.0).amax(1, keepdim=True)
                far = far + 2.0 ** -22 * (1 + 1.5 * torch.where(sees, logits.abs(), 0.0).amax(1, keepdim=True)) + (n / 16 + 200) * 2.0 ** -24
                v, tiny = (x[1] - z[1]).abs(), w.clamp(max=2.0 ** -25)
                t = 2.0 ** -11 * (2 * o.abs() + w @ v) + tiny @ v + tiny.sum(1, keepdim=True) * o.abs() + far * size + 2.0 ** -25
                seen = sees.any(1, keepdim=True)
                out[token:token + new, h * group:(h + 1) * group] = torch.where(seen, o, 0.0).reshape(new, group, 128)
                tol[token:token + new, h * group:(h + 1) * group] = torch.where(seen, t, 0.0).reshape(new, group, 128)
        token += new
    return out, tol


def check(specs, q, starts, lens, news, layer=1, window=0, sinks=0, gone=(), hints=(False, True), step=False, **kw):
    want, tol = definition(specs, kw.pop("q_in", q), lens, news, layer, window, sinks, gone)
    call = kv.batch_chunk_f16 if specs["kv_data"].dtype == torch.float16 else kv.batch_chunk_i4
    results = []
    for hint in hints:
        o = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV)
        given = {"max_new_len": max(news), "max_seq_len": max(lens)} if hint else {}
        assert call(o, q, **specs, layer_idx=layer, seqlen_indptr=None if step else starts, window=window, sinks=sinks, **given, **kw) is None
        off = (o.double() - want).abs()
        assert bool((off <= tol).all()), f"hint {hint}: {float((off / tol.clamp(min=1e-30)).max())} of what is allowed, at {(off - tol).argmax().item()}"
        results.append(o)
    return results


SHAPES = [                                                  # page size, tokens held, new ones
    (16, [5], [5]), (16, [1], [1]), (16, [17, 64, 1], [1, 64, 1]), (16, [208], [5]), (16, [700, 33, 129], [3, 33, 100]),
    (64, [64, 1000, 63], [64, 7, 2]), (128, [300, 128], [257, 1]), (5, [11, 1, 64], [3, 1, 40]), (7, [200, 20], [150, 20]),
    (48, [500], [90]), (2048, [2048, 31], [9, 31]), (1, [40], [12]), (16, [40, 0, 9, 30], [4, 0, 0, 30]),
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,group", [(4, 1), (2, 8), (3, 3), (1, 5)])
@pytest.mark.parametrize("page_size,lens,news", SHAPES)
def test_chunks_of_all_lengths(page_size, lens, news, heads, group, f16):
    specs, q, starts = make(page_size * 7 + len(lens), page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (33, 0), (100, 40), (64, 1000), (5000, 3)])
@pytest.mark.parametrize("page_size,lens,news,heads,group", [
    (16, [700, 33, 129], [90, 33, 1], 2, 4), (5, [64, 300], [64, 20], 3, 1), (64, [1500], [200], 1, 8)])
def test_windows_and_sinks(page_size, lens, news, heads, group, window, sinks, f16):
    specs, q, starts = make(window + sinks, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (128, 4), (1000, 16)])
@pytest.mark.parametrize("page_size,lens,heads,group", [(16, [1, 500, 4001], 4, 1), (32, [3000] * 2, 2, 8), (7, [90, 1000], 5, 2), (128, [9000], 1, 16)])
def test_one_token_per_sequence(page_size, lens, heads, group, window, sinks, f16):
    """The serving step, without bounds of new tokens, whole and split along the positions."""
    news = [1] * len(lens)
    specs, q, starts = make(page_size + window, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks, step=True)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


def scale_values(specs, seed):
    """Values' parameters times powers of two from 2^-20 to 2^11."""
    e = torch.randint(-20, 12, specs["kv_param"].shape[:-1], generator=torch.Generator().manual_seed(seed)).to(DEV)
    specs["kv_param"][:, :, 1] *= torch.exp2(e.double()).half()[:, :, 1, ..., None]


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("news", [[40, 90], [10, 20]])
@pytest.mark.parametrize("f16", [False, True])
def test_large_logits_and_scales(f16, news, seed):
    """Softmaxes that a few positions decide, running maxima that grow by hundreds, and scales from 2^-24 to 2^10."""
    lens = [600, 90]
    specs, q, starts = make(5 + seed, 16, lens, news, 2, 2, f16, spread=12.0)
    check(specs, q, starts, lens, news)
    if not f16:
        scale_values(specs, seed)
        check(specs, q, starts, lens, news)


def test_scales_that_are_zero_or_negative():
    """kv_param is the caller's: a scale of zero leaves the zero point alone, a negative one turns the codes round."""
    lens, news = [100], [60]
    specs, q, starts = make(6, 16, lens, news, 2, 1)
    specs["kv_param"][:, :, :, :, ::3, 0] = 0
    specs["kv_param"][:, :, :, :, 1::3, 0] *= -1
    check(specs, q, starts, lens, news)


@pytest.mark.parametrize("f16", [False, True])
def test_rows_that_see_nothing_are_zero_and_rows_of_no_sequence_are_left(f16):
    """A sequence without pages, one with fewer tokens than new ones, and rows before the first and behind the last bound."""
    lens, news = [0, 3, 20], [4, 7, 5]
    specs, q, starts = make(8, 16, lens, news, 2, 2, f16)
    check(specs, q, starts, lens, news)
    wide = torch.cat([q, q, q[:9]])                        # bounds 16 .. 32 of 41
    want, tol = definition(specs, q, lens, news, 1)
    for hint in ({}, {"max_new_len": 7, "max_seq_len": 20}, {"max_new_len": 1, "max_seq_len": 4000}):
        o = torch.full(wide.shape, 7.0, dtype=torch.float16, device=DEV)
        call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
        call(o, wide, **specs, layer_idx=1, seqlen_indptr=starts + 16, **hint)
        assert bool((o[:16] == 7).all()) and bool((o[32:] == 7).all())
        assert bool(((o[16:32].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size", [16, 6])
def test_page_numbers_outside_the_pool_are_skipped(page_size, f16):
    lens, news = [50, 90], [20, 30]
    specs, q, starts = make(9, page_size, lens, news, 2, 2, f16)
    at = int(specs["kv_indptr"][1])
    specs["kv_indices"][1], specs["kv_indices"][at + 2] = specs["kv_data"].shape[0], -5
    gone = [(0, p) for p in range(page_size, 2 * page_size)] + [(1, p) for p in range(2 * page_size, 3 * page_size)]
    check(specs, q, starts, lens, news, gone=gone)


@pytest.mark.parametrize("f16", [False, True])
def test_strided_queries_and_outputs(f16):
    """q and o as slices of wider rows: what lies beside them is left as it is."""
    lens, news = [70, 30], [33, 30]
    specs, q, starts = make(10, 16, lens, news, 2, 4, f16, fused=512)
    assert q.stride(0) == 8 * 128 + 512
    want, tol = definition(specs, q, lens, news, 1)
    rows = torch.full((q.shape[0], 8 * 128 + 64), 3.0, dtype=torch.float16, device=DEV)
    o = rows[:, :1024].view(q.shape)
    (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **specs, layer_idx=1, seqlen_indptr=starts)
    assert bool(((o.double() - want).abs() <= tol).all()) and bool((rows[:, 1024:] == 3).all())


@pytest.mark.parametrize("f16", [False, True])
def test_query_transform_inside(f16):
    """q_hadamard: matmul_had_cuda of the query, whose fp16 values may differ by a step where 32-bit sums do: every one of 128 terms of a
    logit by u |q| |k|, hence the logits by u sum |q_i k_i| / sqrt(128) -- added to the tolerance as an error of the weights."""
    lens, news = [200, 60], [37, 1]
    specs, q, starts = make(11, 16, lens, news, 2, 3, f16)
    qh = kv.matmul_had_cuda(q.contiguous(), torch.float16)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    want, tol = definition(specs, qh, lens, news, 1)
    o = torch.empty_like(qh)
    call(o, q, **specs, layer_idx=1, seqlen_indptr=starts, q_hadamard=True)
    apart = torch.empty_like(qh)
    call(apart, qh, **specs, layer_idx=1, seqlen_indptr=starts)
    biggest = float(specs["kv_data"].abs().nan_to_num().amax()) if f16 else 0.55 * 15
    more = 2.0 ** -11 * 2 * qh.double().abs().sum(-1, keepdim=True) * biggest / math.sqrt(128) * biggest
    assert bool(((apart.double() - want).abs() <= tol).all())
    assert bool(((o.double() - want).abs() <= tol + more).all())
    assert float((o - apart).double().norm() / apart.double().norm()) < 2.0 ** -10


def test_wrong_hints_cost_time_only():
    lens, news = [300, 50], [120, 50]
    specs, q, starts = make(12, 16, lens, news, 2, 2)
    want, tol = definition(specs, q, lens, news, 1)
    for new, most in ((1, 0), (1, 10), (7, 100000), (100000, 16), (0, 300)):
        o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        kv.batch_chunk_i4(o, q, **specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=most)
        assert bool(((o.double() - want).abs() <= tol).all()), (new, most)


def test_workspace_of_the_caller_and_two_streams():
    """A workspace with arbitrary contents, too small or none, and two streams at work at once, each with its own."""
    lens, news = [5000], [1]
    specs, q, starts = make(13, 16, lens, news, 2, 4)
    want, tol = definition(specs, q, lens, news, 1)
    for size in (1 << 22, 64):
        ws = torch.full((size,), 255, dtype=torch.uint8, device=DEV)
        o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        kv.batch_chunk_i4(o, q, **specs, layer_idx=1, max_seq_len=5000, workspace=ws)
        assert bool(((o.double() - want).abs() <= tol).all())
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            outs.append(torch.empty(q.shape, dtype=torch.float16, device=DEV))
            kv.batch_chunk_i4(outs[-1], q, **specs, layer_idx=1, max_seq_len=5000)
    torch.cuda.synchronize()
    for o in outs:
        assert bool(((o.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("new", [1, 40])
def test_captured_and_replayed(new):
    """A captured call, replayed with other queries in the same memory, eager work between: bit for bit the eager results."""
    lens, news = [3000, 1500], [new, new]
    specs, q, starts = make(14, 16, lens, news, 2, 4)
    args = dict(**specs, layer_idx=1, seqlen_indptr=starts, max_new_len=new, max_seq_len=3000)
    other, o = torch.randn_like(q), torch.empty(q.shape, dtype=torch.float16, device=DEV)
    kv.batch_chunk_i4(o, q, **args)                        # (loads the library's kernels before the capture)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    buffer = q.clone()
    with torch.cuda.graph(graph):
        kv.batch_chunk_i4(o, buffer, **args)
    for k in range(4):
        now = (q, other)[k % 2]
        eager = torch.empty_like(o)
        kv.batch_chunk_i4(eager, now, **args)
        buffer.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eager)


def test_a_call_twice_gives_the_same_bits():
    lens, news = [2000, 700], [300, 1]
    specs, q, starts = make(15, 16, lens, news, 2, 4)
    first, second = (torch.empty(q.shape, dtype=torch.float16, device=DEV) for _ in range(2))
    for o in (first, second):
        kv.batch_chunk_i4(o, q, **specs, layer_idx=1, seqlen_indptr=starts, max_new_len=300, max_seq_len=2000)
    assert torch.equal(first, second)


def test_appended_in_pieces_and_attended_like_single_steps():
    """quantize_append_kv_i4 in two ragged pieces, then the chunk: the outputs of its last tokens are those of batch_decode_i4."""
    heads, page, lens, news = 3, 16, [70, 33], [25, 33]
    specs, q, starts = make(16, page, lens, news, heads, 1, layers=1, spare=0)
    k, v = (torch.randn(sum(news), heads, 128, device=DEV).half() for _ in range(2))
    kv.quantize_append_kv_i4(**specs, k=k, v=v, seqlen_indptr=starts, layer_idx=0)
    o, one = torch.empty_like(q), torch.empty(2, heads, 128, dtype=torch.float16, device=DEV)
    kv.batch_chunk_i4(o, q, **specs, layer_idx=0, seqlen_indptr=starts)
    ends = (starts[1:] - 1).long()
    kv.batch_decode_i4(one, q[ends].contiguous(), **specs, layer_idx=0)
    want, tol = definition(specs, q, lens, news, 0)
    assert bool(((o.double() - want).abs() <= tol).all())
    assert torch.allclose(o[ends], one, rtol=1e-3, atol=1e-3)


def test_refusals():
    specs, q, starts = make(17, 16, [20, 5], [3, 2], 2, 2)
    o = torch.empty_like(q)
    run = lambda **kw: kv.batch_chunk_i4(**{"o": o, "q": q, **specs, "layer_idx": 1, "seqlen_indptr": starts, **kw})
    run()
    for match, kw in (("fp16", {"q": q.float()}), ("3D", {"o": o[0]}), ("contiguous heads", {"q": q.transpose(0, 1).contiguous().transpose(0, 1)}),
                      ("o.size", {"o": torch.empty(4, 4, 128, dtype=torch.float16, device=DEV)}), ("multiple of the cache", {"q": q[:, :3].contiguous(), "o": o[:, :3].contiguous()}),
                      ("one token per sequence", {"seqlen_indptr": None}), ("seqlen_indptr", {"seqlen_indptr": starts.long()}),
                      ("seqlen_indptr", {"seqlen_indptr": starts[:2]}), ("layer_idx", {"layer_idx": 2}), ("negative", {"window": -1}), ("negative", {"sinks": -1}),
                      ("negative", {"max_seq_len": -1}), ("CUDA", {"q": q.cpu()}), ("uint8", {"kv_data": specs["kv_data"].half()}),
                      ("batch_size", {"kv_indptr": specs["kv_indptr"][:2]}), ("overlap", {"q": q[:1].expand(5, 4, 128)})):
        with pytest.raises(RuntimeError, match=match):
            run(**kw)
    with pytest.raises(RuntimeError, match="fp16"):
        kv.batch_chunk_f16(o, q, **specs, layer_idx=1, seqlen_indptr=starts)
    empty = q[:0]
    kv.batch_chunk_i4(empty, empty, **specs, layer_idx=1, seqlen_indptr=starts * 0)          # no new tokens: nothing to do


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,lens,news,heads,group,window,sinks", [
    (16, [600], [600], 2, 1, 0, 0), (16, [1500, 300, 2], [257, 300, 2], 1, 4, 0, 0), (64, [2000], [700], 2, 3, 0, 0), (5, [900], [400], 1, 2, 0, 0),
    (7, [400, 90], [300, 0], 1, 1, 100, 4), (16, [3000], [513], 1, 5, 500, 70), (128, [1000, 1000], [40, 999], 1, 8, 64, 1), (2, [300], [290], 1, 1, 33, 0),
    (1, [200], [200], 1, 2, 0, 0), (16, [70, 5], [200, 9], 2, 2, 0, 0),
])
def test_many_rows(page_size, lens, news, heads, group, window, sinks, f16):
    """Tiles of 256 rows: several of them, rows and positions that fill none, sequences with more new tokens than they hold."""
    specs, q, starts = make(page_size + heads, page_size, lens, news, heads, group, f16)
    check(specs, q, starts, lens, news, window=window, sinks=sinks)


def test_many_rows_large_logits_scales_and_missing_pages():
    lens, news = [700], [400]
    specs, q, starts = make(21, 16, lens, news, 1, 2, spread=12.0)
    check(specs, q, starts, lens, news)
    scale_values(specs, 21)
    specs["kv_param"][:, :, 1, :, ::5, 0] = 0
    specs["kv_param"][:, :, 1, :, 1::5, 0] *= -1
    check(specs, q, starts, lens, news)
    specs["kv_indices"][3], specs["kv_indices"][20] = -1, 1 << 30
    check(specs, q, starts, lens, news, gone=[(0, p) for p in [*range(48, 64), *range(320, 336)]])


@pytest.mark.parametrize("f16", [False, True])
def test_many_rows_with_the_transform_inside(f16):
    lens, news = [500], [300]
    specs, q, starts = make(22, 16, lens, news, 1, 2, f16)
    qh = kv.matmul_had_cuda(q.contiguous(), torch.float16)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    apart, o = torch.empty_like(qh), torch.empty_like(qh)
    call(apart, qh, **specs, layer_idx=1, seqlen_indptr=starts)
    call(o, q, **specs, layer_idx=1, seqlen_indptr=starts, q_hadamard=True)
    assert float((o - apart).double().norm() / apart.double().norm()) < 2.0 ** -10


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("lens,news,heads,group,window,sinks", [([70], [40], 2, 1, 0, 0), ([90, 33], [30, 33], 1, 4, 20, 3), ([300], [1], 2, 3, 100, 2),
                                                                ([600], [400], 1, 2, 0, 0), ([900], [500], 1, 1, 70, 5)])
def test_infinities_and_nans_reach_only_rows_that_see_them(lens, news, heads, group, window, sinks, f16):
    """A key or a value that is no number, or infinite, at a position that some rows do not see (later, outside the window): those rows' results are as if
    it were any other, bit for bit; a row that sees one of them is not finite in the dimensions concerned."""
    specs, q, starts = make(30 + sum(lens), 16, lens, news, heads, group, f16)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    page = lambda b, pos: int(specs["kv_indices"][int(specs["kv_indptr"][b]) + pos // 16])
    at = [(0, lens[0] - 2, 1), (0, lens[0] - 5, 0), (0, 1, 1), (0, lens[0] - news[0], 1), (len(lens) - 1, lens[-1] - 1, 1), (0, lens[0] // 2, 1)]
    clean = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    call(clean, q, **specs, layer_idx=1, seqlen_indptr=starts, window=window, sinks=sinks)
    for k, (b, pos, side) in enumerate(at):
        bad = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
        value = (float("inf"), float("nan"), -float("inf"))[k % 3]
        if f16:
            bad["kv_data"][page(b, pos), 1, side, :, pos % 16, 5::40] = value
        else:
            bad["kv_param"][page(b, pos), 1, side, :, pos % 16, k % 2] = value
        o = torch.full_like(clean, 9.0)
        call(o, q, **bad, layer_idx=1, seqlen_indptr=starts, window=window, sinks=sinks)
        first = sum(news[:b])
        for t in range(q.shape[0]):
            place = lens[b] - news[b] + t - first
            sees = first <= t < first + news[b] and pos <= place and (not window or place - pos < window or pos < sinks)
            if not sees:
                assert torch.equal(o[t], clean[t]), (k, t)
            elif side == 1 and f16:
                assert not bool(torch.isfinite(o[t, :, 5::40]).any()), (k, t)
                rest = torch.ones(128, dtype=torch.bool)
                rest[5::40] = False
                assert torch.equal(o[t][:, rest], clean[t][:, rest]), (k, t)
            elif side == 1:
                assert not bool(torch.isfinite(o[t]).any()), (k, t)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("batch,most,group", [(64, 40, 4), (65, 40, 4), (70, 70, 8), (130, 3, 8)])
def test_many_sequences(batch, most, group, f16):
    """Ragged batches whose work items are counted (64 sequences) and are not (more), sequences without new tokens among them."""
    news = [(7 * b) % (most + 1) for b in range(batch)]
    lens = [n + (13 * b) % 90 for b, n in enumerate(news)]
    specs, q, starts = make(batch, 16, lens, news, 2, group, f16)
    check(specs, q, starts, lens, news)
    check(specs, q, starts, lens, news, window=30, sinks=3)

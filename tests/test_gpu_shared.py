"""Attention of sequences that share a prefix (batch_shared_i4, batch_shared_f16) against its definition in 64 bits: a softmax over the prefix and the
sequence's own positions.  The tolerance is that of attention of new tokens (test_gpu_chunk.py): a row's states of both launches are joined in
32 bits, and in each the smallest weights are rounded in units of its own largest one, which is no larger than the row's.

The logarithm of a row's sum: a weight counts as rounded, w_j (1 + d_j) with |d_j| <= 2^-11 (2^-25 of the largest where it is smaller), so the sum is off by
as much, relatively, and its logarithm by 2^-11 + n 2^-25 at most; a logit's error moves it by no more than itself; the sum's additions and the
logarithm itself are in fp32, 2^-21 of what they give and a few steps of it."""
import gc
import math

import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, make, scale_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def make_shared(seed, page_size, prefixes, members, lens, news, heads, group, f16=False, **kw):
    """A cache whose last page lists are the prefixes': (specs, prefix arguments, q, bounds)."""
    specs, q, starts = make(seed, page_size, [*lens, *prefixes], [*news, *([0] * len(prefixes))], heads, group, f16, **kw)
    n = len(lens)
    prefix = {"prefix_indptr": specs["kv_indptr"][n:].contiguous(), "prefix_indices": specs["kv_indices"], "prefix_last_page_offset": specs["last_page_offset"][n:].contiguous(),
              "prefix_sequences": None if members is None else torch.tensor(members, dtype=torch.int32, device=DEV)}
    specs = {**specs, "kv_indptr": specs["kv_indptr"][:n + 1].contiguous(), "last_page_offset": specs["last_page_offset"][:n].contiguous()}
    return specs, prefix, q, starts[:n + 1].contiguous()


def vectors(specs, indptr, i, n, layer, h):
    """(scale code, zero) of the keys and of the values of list i, its first n positions, in 64 bits."""
    data, param = specs["kv_data"], specs["kv_param"]
    lo, hi = indptr[i:i + 2].tolist()
    held = specs["kv_indices"][lo:hi].long()
    out = []
    for side in (0, 1):
        rows = data[held, layer, side, h].reshape(-1, data.shape[-1])[:n]
        if data.dtype == torch.float16:
            out.append((rows.double(), torch.zeros(n, 1, dtype=torch.float64, device=DEV)))
        else:
            pr = param[held, layer, side, h].reshape(-1, 2)[:n].double()
            out.append((pr[:, :1] * torch.stack([rows & 15, rows >> 4], -1).reshape(n, 128).double(), pr[:, 1:]))
    return out


def definition(specs, prefix, q, prefixes, members, lens, news, layer):
    """(outputs, how far off), (logarithms, how far off)"""
    heads, n_seq = specs["kv_data"].shape[3], len(lens)
    group = q.shape[1] // heads
    out, tol = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    lse, lse_tol = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=DEV), torch.zeros(q.shape[:2], dtype=torch.float64, device=DEV)
    members = [0, n_seq] if members is None else members
    token = 0
    for b, (n, new) in enumerate(zip(lens, news)):
        of = [p for p in range(len(prefixes)) if members[p] <= b < members[p + 1]]
        before = prefixes[of[0]] if of else 0
        if new and n + before:
            place = torch.arange(n - new, n, device=DEV)[:, None].repeat(1, group).reshape(-1, 1)
            sees = torch.cat([torch.ones(new * group, before, dtype=torch.bool, device=DEV), torch.arange(n, device=DEV)[None] <= place], 1)
            for h in range(heads):
                parts = ([vectors(specs, prefix["prefix_indptr"], of[0], before, layer, h)] if before else []) + ([vectors(specs, specs["kv_indptr"], b, n, layer, h)] if n else [])
                (xk, zk), (xv, zv) = ((torch.cat([p[side][0] for p in parts]), torch.cat([p[side][1] for p in parts])) for side in (0, 1))
                qs = q[token:token + new, h * group:(h + 1) * group].reshape(-1, 128).double()
                logits = (qs @ xk.T - qs.sum(1, keepdim=True) * zk.T) / math.sqrt(128)
                terms = (qs.abs() @ xk.abs().T + qs.abs().sum(1, keepdim=True) * zk.abs().T) / math.sqrt(128)
                masked = torch.where(sees, logits, -math.inf)
                w = torch.where(sees, torch.softmax(masked.nan_to_num(nan=0.0, neginf=-1e300), 1), 0.0)
                o, size = w @ (xv - zv), w @ (xv.abs() + zv.abs())
                small = 2.0 ** -21 * xk.abs().sum(1)[None] / math.sqrt(128)
                logit_off = torch.where(sees, 140 * 2.0 ** -24 * terms + small, 0.0).amax(1, keepdim=True)
                biggest = torch.where(sees, logits.abs(), 0.0).amax(1, keepdim=True)
                far = 2 * logit_off + 2.0 ** -22 * (1 + 1.5 * biggest) + ((n + before) / 16 + 200) * 2.0 ** -24
                v, tiny = (xv - zv).abs(), w.clamp(max=2.0 ** -25)
                t = 2.0 ** -11 * (2 * o.abs() + w @ v) + tiny @ v + tiny.sum(1, keepdim=True) * o.abs() + far * size + 2.0 ** -25
                seen = sees.any(1, keepdim=True)
                at = (slice(token, token + new), slice(h * group, (h + 1) * group))
                out[at], tol[at] = torch.where(seen, o, 0.0).reshape(new, group, 128), torch.where(seen, t, 0.0).reshape(new, group, 128)
                lse[at] = torch.logsumexp(masked, 1).reshape(new, group)
                lse_tol[at] = (2.0 ** -11 + tiny.sum(1, keepdim=True) + far + 2.0 ** -21 * (1 + 2 * biggest)).reshape(new, group)
        token += new
    return (out, tol), (lse, lse_tol)


def check_lse(lse, want, tol):
    seen = want > -math.inf
    assert bool((lse[~seen] == -math.inf).all())
    off = (lse.double() - want).abs()[seen]
    assert bool((off <= tol[seen]).all()), f"{float((off / tol[seen]).max())} of what is allowed"


def check(specs, prefix, q, starts, prefixes, members, lens, news, layer=1, step=False, hints=(False, True), **kw):
    (want, tol), (lse_want, lse_tol) = definition(specs, prefix, q, prefixes, members, lens, news, layer)
    call = kv.batch_shared_f16 if specs["kv_data"].dtype == torch.float16 else kv.batch_shared_i4
    results = []
    for hint in hints:
        o, lse = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV), torch.full(q.shape[:2], float("nan"), device=DEV)
        given = {"max_new_len": max(news), "max_seq_len": max(lens), "max_prefix_len": max(prefixes)} if hint else {}
        assert call(o, q, **specs, layer_idx=layer, **prefix, seqlen_indptr=None if step else starts, lse=lse if hint else None, **given, **kw) is None
        off = (o.double() - want).abs()
        assert bool((off <= tol).all()), f"hint {hint}: {float((off / tol.clamp(min=1e-30)).max())} of what is allowed, at {(off - tol).argmax().item()}"
        if hint:
            check_lse(lse, lse_want, lse_tol)
        results.append(o)
    return results


SHAPES = [                                                  # page size, prefixes, first sequences, own tokens, new ones
    (16, [1], None, [1], [1]), (16, [33], None, [5, 1, 18], [1, 1, 1]), (16, [700], None, [3, 40, 17, 1], [3, 5, 1, 1]), (64, [1000], None, [64, 70], [64, 2]),
    (7, [150], None, [20, 1], [13, 1]), (16, [90, 33, 300], [0, 2, 3, 5], [9, 1, 30, 20, 2], [4, 1, 2, 20, 1]), (1, [40], None, [12, 3], [5, 3]),
    (128, [64, 128], [0, 1, 4], [130, 1, 5, 9], [100, 1, 2, 9]), (48, [500], None, [90], [90]), (5, [64, 3], [0, 1, 2], [2, 30], [2, 11]),
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,group", [(4, 1), (2, 8), (3, 3)])
@pytest.mark.parametrize("page_size,prefixes,members,lens,news", SHAPES)
def test_prefixes_of_all_lengths(page_size, prefixes, members, lens, news, heads, group, f16):
    specs, prefix, q, starts = make_shared(page_size * 7 + len(lens), page_size, prefixes, members, lens, news, heads, group, f16)
    check(specs, prefix, q, starts, prefixes, members, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,prefixes,members,lens,heads,group", [
    (16, [4000], None, [1, 30, 500], 4, 1), (16, [5000], None, list(range(1, 41)), 2, 8), (32, [300, 3000], [0, 10, 33], [7] * 33, 2, 4), (7, [900], None, [90, 1000], 5, 2),
    (128, [9000], None, [1], 1, 16), (16, [2000], None, [3000], 2, 4)])
def test_one_token_per_sequence(page_size, prefixes, members, lens, heads, group, f16):
    news = [1] * len(lens)
    specs, prefix, q, starts = make_shared(page_size + len(lens), page_size, prefixes, members, lens, news, heads, group, f16)
    check(specs, prefix, q, starts, prefixes, members, lens, news, step=True)
    check(specs, prefix, q, starts, prefixes, members, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,prefixes,members,lens,news,heads,group", [
    (16, [3000], None, [400, 300], [400, 300], 2, 2), (64, [1500, 700], [0, 1, 3], [257, 30, 300], [257, 30, 256], 1, 4), (5, [500], None, [300, 1], [200, 1], 1, 3)])
def test_many_rows(page_size, prefixes, members, lens, news, heads, group, f16):
    """The prefix goes to tiles of 256 rows, the sequences' own positions too."""
    specs, prefix, q, starts = make_shared(page_size + heads, page_size, prefixes, members, lens, news, heads, group, f16)
    check(specs, prefix, q, starts, prefixes, members, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,prefix_len,members,lens,news,heads,group", [
    (16, 8000, None, [70] * 9, [70] * 9, 5, 2),              # five tiles a head: no number of shares goes into them, nor they into it
    (16, 900, None, [130] * 20, [130] * 20, 3, 8),           # more tiles than shares
    (64, 20000, None, [300], [300], 1, 1),                   # more shares than a tile has states
    (16, 40, None, [300, 90], [300, 90], 2, 4),              # a step of the prefix for several tiles
    (7, 3000, [0, 2], [200, 100, 300], [200, 100, 300], 2, 3),              # sequences behind the prefix's last: tiles without rows
    (16, 2000, [1, 1], [200, 300], [200, 300], 2, 2),        # a prefix of no sequence
    (16, 0, None, [300, 100], [300, 100], 2, 2)])            # and one without positions
def test_one_prefix_and_many_rows(page_size, prefix_len, members, lens, news, heads, group, f16):
    """The steps of a prefix's tiles dealt out evenly: shares that begin and end inside tiles, whatever is hinted."""
    specs, prefix, q, starts = make_shared(prefix_len + heads, page_size, [prefix_len], members, lens, news, heads, group, f16)
    outs = check(specs, prefix, q, starts, [prefix_len], members, lens, news)
    (want, tol), _ = definition(specs, prefix, q, [prefix_len], members, lens, news, 1)
    call = kv.batch_shared_f16 if f16 else kv.batch_shared_i4
    for hint in (1, 500, 3 * prefix_len, 1 << 40):
        o = torch.empty_like(outs[0])
        call(o, q, **specs, layer_idx=1, **prefix, seqlen_indptr=starts, max_new_len=max(news), max_seq_len=max(lens), max_prefix_len=hint,
             workspace=torch.full((1 << 28,), 255, dtype=torch.uint8, device=DEV))
        assert bool(((o.double() - want).abs() <= tol).all()), hint


@pytest.mark.parametrize("news", [[1, 1, 1, 1, 1], [3, 0, 200, 1, 9]])
@pytest.mark.parametrize("f16", [False, True])
def test_sequences_without_a_prefix_empty_prefixes_and_empty_sequences(f16, news):
    """Sequences before the first bound and behind the last one, prefixes without positions or without sequences, sequences without positions of their own."""
    prefixes, members = [50, 0, 20, 700], [1, 2, 3, 3, 4]
    lens = [max(3, n) for n in news]
    lens[1] = 0
    specs, prefix, q, starts = make_shared(3, 16, prefixes, members, lens, news, 2, 2, f16)
    check(specs, prefix, q, starts, prefixes, members, lens, news)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("news", [[1] * 6, [50, 1, 30, 7, 90, 2]])
def test_large_logits_and_scales(f16, news):
    """Rows that the prefix alone decides, or their own positions alone."""
    prefixes, lens = [300], [n + 9 for n in news]
    specs, prefix, q, starts = make_shared(5, 16, prefixes, None, lens, news, 2, 4, f16, spread=12.0)
    check(specs, prefix, q, starts, prefixes, None, lens, news)
    if not f16:
        scale_values(specs, 5)
        check(specs, prefix, q, starts, prefixes, None, lens, news)


@pytest.mark.parametrize("f16", [False, True])
def test_no_difference_from_pages_of_every_sequence(f16):
    """A prefix of whole pages, also as the first pages of every sequence: the same outputs within both calls' roundings."""
    page, prefixes, lens, news = 16, [320], [30, 7, 64], [5, 7, 1]
    specs, prefix, q, starts = make_shared(6, page, prefixes, None, lens, news, 2, 3, f16)
    (want, tol), _ = definition(specs, prefix, q, prefixes, None, lens, news, 1)
    bounds, shared = specs["kv_indptr"].tolist(), specs["kv_indices"][prefix["prefix_indptr"][0]:prefix["prefix_indptr"][1]]
    whole = torch.cat([torch.cat([shared, specs["kv_indices"][bounds[b]:bounds[b + 1]]]) for b in range(3)])
    indptr = specs["kv_indptr"] + 20 * torch.arange(4, dtype=torch.int32, device=DEV)
    o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **{**specs, "kv_indices": whole, "kv_indptr": indptr}, layer_idx=1, seqlen_indptr=starts)
    assert bool(((o.double() - want).abs() <= tol).all())
    check(specs, prefix, q, starts, prefixes, None, lens, news)


@pytest.mark.parametrize("f16", [False, True])
def test_rows_of_no_sequence_strides_and_the_transform(f16):
    """q and o slices of wider rows; rows before and behind the bounds are left; q_hadamard is matmul_had_cuda's."""
    prefixes, lens, news = [200], [20, 30], [4, 9]
    specs, prefix, q, starts = make_shared(8, 16, prefixes, None, lens, news, 2, 2, f16, fused=256)
    assert q.stride(0) == 4 * 128 + 256
    call = kv.batch_shared_f16 if f16 else kv.batch_shared_i4
    wide = torch.cat([q, q, q])
    (want, tol), (lse_want, lse_tol) = definition(specs, prefix, q, prefixes, None, lens, news, 1)
    rows, lse = torch.full((wide.shape[0], 4 * 128 + 64), 7.0, dtype=torch.float16, device=DEV), torch.full((wide.shape[0], 4), 7.0, device=DEV)
    o = rows[:, :512].view(wide.shape)
    call(o, wide, **specs, layer_idx=1, **prefix, seqlen_indptr=starts + 13, lse=lse, max_seq_len=30, max_prefix_len=200)
    assert bool((o[:13] == 7).all()) and bool((o[26:] == 7).all()) and bool((rows[:, 512:] == 7).all())
    assert bool((lse[:13] == 7).all()) and bool((lse[26:] == 7).all())
    assert bool(((o[13:26].double() - want).abs() <= tol).all())
    check_lse(lse[13:26], lse_want, lse_tol)
    inside, apart = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape, dtype=torch.float16, device=DEV)
    call(inside, q, **specs, layer_idx=1, **prefix, seqlen_indptr=starts, q_hadamard=True)
    call(apart, kv.matmul_had_cuda(q.contiguous(), torch.float16), **specs, layer_idx=1, **prefix, seqlen_indptr=starts)
    assert float((inside - apart).double().norm() / apart.double().norm()) < 2.0 ** -10


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("lens,news,window,sinks,step", [([300, 20], [40, 3], 0, 0, False), ([5000], [1], 0, 0, True), ([700], [600], 0, 0, False), ([900, 33], [100, 1], 64, 4, False)])
def test_logarithms_without_a_prefix(lens, news, window, sinks, step, f16):
    """batch_chunk's lse, whole and split, and its outputs, which are what they are without it."""
    specs, q, starts = make(9, 16, lens, news, 2, 4, f16)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    for hint in ({}, {"max_new_len": max(news), "max_seq_len": max(lens)}):
        o, alone, lse = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape[:2], device=DEV)
        given = dict(**specs, layer_idx=1, seqlen_indptr=None if step else starts, window=window, sinks=sinks, **hint)
        call(o, q, **given, lse=lse)
        call(alone, q, **given)
        assert float((o - alone).double().norm()) <= 2.0 ** -11 * float(alone.double().norm())
        token = 0
        for b, (n, new) in enumerate(zip(lens, news)):
            for h in range(2):
                (xk, zk), _ = vectors(specs, specs["kv_indptr"], b, n, 1, h)
                qs = q[token:token + new, 4 * h:4 * h + 4].reshape(-1, 128).double()
                place, j = torch.arange(n - new, n, device=DEV)[:, None].repeat(1, 4).reshape(-1, 1), torch.arange(n, device=DEV)[None]
                sees = (j <= place) & ((place - j < window) | (j < sinks) if window else True)
                logits = torch.where(sees, (qs @ xk.T - qs.sum(1, keepdim=True) * zk.T) / math.sqrt(128), -math.inf)
                terms = ((qs.abs() @ xk.abs().T + qs.abs().sum(1, keepdim=True) * zk.abs().T) / math.sqrt(128)).amax(1)
                want = torch.logsumexp(logits, 1)
                tol = 2.0 ** -11 + n * 2.0 ** -25 + 140 * 2.0 ** -24 * terms + 2.0 ** -21 * xk.abs().sum(1).amax() / math.sqrt(128) + 2.0 ** -20 * (1 + want.abs())
                assert bool(((lse[token:token + new, 4 * h:4 * h + 4].reshape(-1).double() - want).abs() <= tol).all())
            token += new


def test_wrong_hints_cost_time_only():
    prefixes, lens, news = [600], [300, 50], [120, 50]
    specs, prefix, q, starts = make_shared(12, 16, prefixes, None, lens, news, 2, 2)
    (want, tol), _ = definition(specs, prefix, q, prefixes, None, lens, news, 1)
    for new, most, long in ((1, 0, 0), (1, 10, 5), (7, 100000, 1 << 40), (100000, 16, 600), (0, 300, 1)):
        o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        kv.batch_shared_i4(o, q, **specs, layer_idx=1, **prefix, seqlen_indptr=starts, max_new_len=new, max_seq_len=most, max_prefix_len=long)
        assert bool(((o.double() - want).abs() <= tol).all()), (new, most, long)


def test_workspaces_streams_and_the_same_bits():
    """A workspace of arbitrary contents, one that is too small, two streams at work at once; a call twice gives the same bits."""
    prefixes, lens, news = [5000], [40, 3, 17], [1, 1, 1]
    specs, prefix, q, starts = make_shared(13, 16, prefixes, None, lens, news, 2, 4)
    args = dict(**specs, layer_idx=1, **prefix, max_seq_len=40, max_prefix_len=5000)
    want = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    kv.batch_shared_i4(want, q, **args)
    for size in (1 << 24, 64):
        o = torch.empty_like(want)
        kv.batch_shared_i4(o, q, **args, workspace=torch.full((size,), 255, dtype=torch.uint8, device=DEV))
        assert torch.equal(o, want)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(2)], []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            outs.append(torch.empty_like(want))
            kv.batch_shared_i4(outs[-1], q, **args)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("new", [1, 60])
def test_captured_and_replayed(new):
    prefixes, lens, news = [2000], [100, 70], [new, new]
    specs, prefix, q, starts = make_shared(14, 16, prefixes, None, lens, news, 2, 4)
    args = dict(**specs, layer_idx=1, **prefix, seqlen_indptr=starts, max_new_len=new, max_seq_len=100, max_prefix_len=2000)
    other, o, lse = torch.randn_like(q), torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape[:2], device=DEV)
    kv.batch_shared_i4(o, q, **args, lse=lse)
    torch.cuda.synchronize()
    graph, buffer = torch.cuda.CUDAGraph(), q.clone()
    with torch.cuda.graph(graph):
        kv.batch_shared_i4(o, buffer, **args, lse=lse)
    for k in range(4):
        now = (q, other)[k % 2]
        eager, eager_lse = torch.empty_like(o), torch.empty_like(lse)
        kv.batch_shared_i4(eager, now, **args, lse=eager_lse)
        buffer.copy_(now)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, eager) and torch.equal(lse, eager_lse)


@pytest.mark.parametrize("f16", [False, True])
def test_page_numbers_outside_the_pool_are_skipped(f16):
    """A prefix page that is none counts as not there: the result is that of a prefix without its positions."""
    prefixes, lens, news = [48], [20, 9], [3, 9]
    specs, prefix, q, starts = make_shared(15, 16, prefixes, None, lens, news, 2, 2, f16)
    call = kv.batch_shared_f16 if f16 else kv.batch_shared_i4
    at = int(prefix["prefix_indptr"][0])
    less = {**prefix, "prefix_indices": torch.cat([prefix["prefix_indices"][:at + 1], prefix["prefix_indices"][at + 2:]]),
            "prefix_indptr": torch.tensor([at, at + 2], dtype=torch.int32, device=DEV)}
    (want, tol), _ = definition({**specs, "kv_indices": less["prefix_indices"]}, less, q, [32], None, lens, news, 1)
    for page in (-1, specs["kv_data"].shape[0], 1 << 30):
        gone = {**prefix, "prefix_indices": prefix["prefix_indices"].clone()}
        gone["prefix_indices"][at + 1] = page
        o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
        call(o, q, **specs, layer_idx=1, **gone, seqlen_indptr=starts)
        assert bool(((o.double() - want).abs() <= tol).all()), page


@pytest.mark.parametrize("f16", [False, True])
def test_infinities_and_nans_of_one_prefix_stay_with_its_sequences(f16):
    prefixes, members, lens, news = [40, 70], [0, 2, 3], [5, 9, 20], [2, 9, 1]
    specs, prefix, q, starts = make_shared(16, 16, prefixes, members, lens, news, 2, 2, f16)
    call = kv.batch_shared_f16 if f16 else kv.batch_shared_i4
    clean, o = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape, dtype=torch.float16, device=DEV)
    call(clean, q, **specs, layer_idx=1, **prefix, seqlen_indptr=starts)
    page = int(specs["kv_indices"][prefix["prefix_indptr"][0]])
    for value in (float("nan"), float("inf")):
        bad = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
        (bad["kv_data"] if f16 else bad["kv_param"])[page, 1, 1, :, 3] = value
        call(o, q, **bad, layer_idx=1, **prefix, seqlen_indptr=starts)
        assert not bool(torch.isfinite(o[:11]).any()) and torch.equal(o[11:], clean[11:])


def test_refusals():
    prefixes, lens, news = [40], [20, 5], [3, 2]
    specs, prefix, q, starts = make_shared(17, 16, prefixes, None, lens, news, 2, 2)
    o, lse = torch.empty(q.shape, dtype=torch.float16, device=DEV), torch.empty(q.shape[:2], device=DEV)
    run = lambda **kw: kv.batch_shared_i4(**{"o": o, "q": q, **specs, "layer_idx": 1, **prefix, "seqlen_indptr": starts, "lse": lse, **kw})
    run()
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    for match, kw in (("prefix_indptr", {"prefix_indptr": None}), ("prefix_indptr", {"prefix_indptr": prefix["prefix_indptr"].long()}),
                      ("prefix_indices", {"prefix_indices": None}), ("prefix_last_page_offset", {"prefix_last_page_offset": None}),
                      ("one entry more", {"prefix_last_page_offset": two}), ("several prefixes", {"prefix_last_page_offset": two, "prefix_indptr": torch.zeros(3, dtype=torch.int32, device=DEV)}),
                      ("prefix_sequences", {"prefix_sequences": two[:1]}), ("prefix_sequences", {"prefix_sequences": two.long()}), ("CUDA", {"prefix_indices": prefix["prefix_indices"].cpu()}),
                      ("lse", {"lse": lse.half()}), ("lse", {"lse": lse[:, :3]}), ("lse", {"lse": lse[:4]}), ("negative", {"max_prefix_len": -1}), ("negative", {"max_seq_len": -1}),
                      ("fp16", {"q": q.float()}), ("multiple of the cache", {"q": q[:, :3].contiguous(), "o": o[:, :3].contiguous()}), ("one token per sequence", {"seqlen_indptr": None}),
                      ("layer_idx", {"layer_idx": 2}), ("batch_size", {"kv_indptr": specs["kv_indptr"][:2]})):
        with pytest.raises(RuntimeError, match=match):
            run(**kw)
    with pytest.raises(TypeError):
        run(window=5)
    with pytest.raises(RuntimeError, match="lse"):
        kv.batch_chunk_i4(o, q, **specs, layer_idx=1, seqlen_indptr=starts, lse=lse.double())
    run(q=q[:0], o=o[:0], lse=lse[:0], seqlen_indptr=starts * 0)

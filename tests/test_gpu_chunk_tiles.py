"""Attention of new tokens over the paged cache at sizes that go to the kernel of 256 rows (some 57000 rows and more in a call: 224 tiles of 256 rows are one turn
of the chip, 1792 of 32 would be several), against the definition in 64 bits and with the tolerances of test_gpu_chunk.py."""
import gc
import math

import pytest
import torch

from quarot_amd import _lib
from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, check, definition, make, scale_values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def lower(specs, q):
    """Keys around one, queries around minus twelve: every logit is near -12 * 128 / sqrt(128) = -136, its spread 3 to 4."""
    side = specs["kv_data"] if specs["kv_data"].dtype == torch.float16 else specs["kv_param"]
    keys = side[:, :, 0].float() * 0.2
    if side is specs["kv_data"]:
        keys += 1
    else:
        keys[..., 1] -= 1                                  # (the zero point is subtracted)
    side[:, :, 0] = keys.half()
    q.copy_((q.float() * 0.5 - 12).half())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("lens,news,heads,group,window,sinks,gone", [
    ([700], [256], 28, 8, 33, 0, 0), ([700], [256], 224, 1, 100, 0, 0), ([500, 300], [100, 156], 28, 8, 20, 0, 0), ([700], [256], 28, 8, 0, 0, 3),
    ([700], [256], 112, 2, 64, 4, 1)])
def test_rows_whose_first_positions_are_hidden_with_logits_far_below_zero(lens, news, heads, group, window, sinks, gone, f16):
    """A row's weights are those of its logits less their maximum, wherever its first visible position lies in its tile."""
    specs, q, starts = make(40 + heads, 16, lens, news, heads, group, f16, layers=1)
    lower(specs, q)
    specs["kv_indices"][:gone] = -1
    check(specs, q, starts, lens, news, layer=0, window=window, sinks=sinks, gone=[(0, p) for p in range(16 * gone)])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("window,sinks,gone", [(0, 0, False), (3500, 0, False), (3500, 4, False), (0, 0, True), (3500, 4, True)])
def test_splits_whose_first_positions_are_hidden_with_logits_far_below_zero(window, sinks, gone, f16):
    """The same where several workgroups share a tile's positions; gone: of every 256 positions 128 are on no page, wherever a workgroup begins."""
    lens, news = [4513], [512]
    specs, q, starts = make(45, 16, lens, news, 32, 1, f16, layers=1)
    lower(specs, q)
    assert _lib.lib().qr_batch_chunk_workspace_bytes(1 if f16 else 0, 512, 32, 32, 1, 512, 4513, window, sinks) > 0
    missing = [p for p in range(4513) if gone and p // 128 % 2 == 0]
    specs["kv_indices"][sorted({p // 16 for p in missing})] = -1
    check(specs, q, starts, lens, news, layer=0, window=window, sinks=sinks, gone=[(0, p) for p in missing], hints=(True,))


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,lens,news,heads,group,window,sinks", [
    (16, [256], [256], 28, 8, 0, 0), (16, [700, 40, 1], [200, 40, 1], 28, 8, 0, 0), (64, [1000], [256], 28, 8, 0, 0), (5, [300], [240], 28, 8, 0, 0),
    (7, [400, 90], [256, 0], 56, 4, 100, 4), (16, [1500], [513], 32, 4, 500, 70), (128, [500, 500], [16, 240], 28, 8, 64, 1), (2, [300], [290], 28, 8, 33, 0),
    (1, [260], [250], 28, 8, 0, 0), (16, [70, 5], [250, 9], 28, 8, 0, 0), (48, [900], [256], 75, 3, 1, 0), (16, [900], [256], 224, 1, 40, 100), (6, [700], [256], 224, 1, 130, 3),
    (2048, [700], [256], 28, 8, 5000, 3), (16, [90] * 70, [32] * 70, 28, 8, 0, 0)])
def test_shapes_windows_and_pages(page_size, lens, news, heads, group, window, sinks, f16):
    specs, q, starts = make(page_size + heads, page_size, lens, news, heads, group, f16, layers=1)
    check(specs, q, starts, lens, news, layer=0, window=window, sinks=sinks)


@pytest.mark.parametrize("f16", [False, True])
def test_large_logits_scales_and_missing_pages(f16):
    lens, news = [700], [256]
    specs, q, starts = make(21, 16, lens, news, 28, 8, f16, spread=12.0)
    check(specs, q, starts, lens, news)
    check(specs, q, starts, lens, news, window=90, sinks=2)
    if not f16:
        scale_values(specs, 21)
        specs["kv_param"][:, :, 1, :, ::5, 0] = 0
        specs["kv_param"][:, :, 1, :, 1::5, 0] *= -1
        check(specs, q, starts, lens, news)
    specs["kv_indices"][0], specs["kv_indices"][3], specs["kv_indices"][20] = 1 << 20, -1, 1 << 30
    check(specs, q, starts, lens, news, gone=[(0, p) for p in [*range(16), *range(48, 64), *range(320, 336)]])


@pytest.mark.parametrize("f16", [False, True])
def test_transform_inside_strides_and_rows_of_no_sequence(f16):
    """Queries and outputs in wider rows, bounds that begin behind the first row and end before the last."""
    lens, news = [500], [256]
    specs, q, starts = make(22, 16, lens, news, 28, 8, f16, layers=1, fused=256)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    plain = q.contiguous()
    qh = kv.matmul_had_cuda(plain, torch.float16)
    want, tol = definition(specs, plain, lens, news, 0)
    wide = torch.full((276, 224 * 128 + 64), 3.0, dtype=torch.float16, device=DEV)
    queries = torch.cat([q.new_full((10, 224, 128), float("nan")), q, q.new_full((10, 224, 128), float("nan"))])
    call(wide[:, :224 * 128].view(276, 224, 128), queries, **specs, layer_idx=0, seqlen_indptr=starts + 10)
    o = wide[10:266, :224 * 128].view(256, 224, 128)
    assert bool(((o.double() - want).abs() <= tol).all())
    assert all(bool((t == 3).all()) for t in (wide[:10], wide[266:], wide[:, 224 * 128:]))
    strided = torch.empty_like(plain)
    call(strided, q, **specs, layer_idx=0, seqlen_indptr=starts)
    assert torch.equal(strided, o)
    apart, inside = torch.empty_like(qh), torch.empty_like(qh)
    call(apart, qh, **specs, layer_idx=0, seqlen_indptr=starts)
    call(inside, q, **specs, layer_idx=0, seqlen_indptr=starts, q_hadamard=True)
    biggest = float(specs["kv_data"].abs().nan_to_num().amax()) if f16 else 0.55 * 15
    want, tol = definition(specs, qh, lens, news, 0)
    more = 2.0 ** -11 * 2 * qh.double().abs().sum(-1, keepdim=True) * biggest / math.sqrt(128) * biggest
    assert bool(((apart.double() - want).abs() <= tol).all()) and bool(((inside.double() - want).abs() <= tol + more).all())


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,group,window,sinks", [(28, 8, 0, 0), (28, 8, 70, 5), (224, 1, 100, 0)])
def test_infinities_and_nans(heads, group, window, sinks, f16):
    """A key or a value that is no number, or infinite: rows that do not see its position are as if it were any other, bit for bit; rows that see such a
    value are not finite in the dimensions concerned; rows that see a key which is no number are not finite at all."""
    lens, news = [400], [256]
    specs, q, starts = make(30 + group, 16, lens, news, heads, group, f16, layers=1)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    clean = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    call(clean, q, **specs, layer_idx=0, seqlen_indptr=starts, window=window, sinks=sinks)
    place = torch.arange(144, 400, device=DEV)
    dims = torch.zeros(128, dtype=torch.bool, device=DEV)
    dims[5::40] = True
    for k, (pos, side, value) in enumerate([(398, 1, "inf"), (395, 0, "nan"), (1, 1, "-inf"), (144, 1, "nan"), (300, 0, "nan"), (200, 1, "inf"), (200, 0, "inf")]):
        bad = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
        at = int(specs["kv_indices"][pos // 16])
        if f16:
            bad["kv_data"][at, 0, side, :, pos % 16, 5::40] = float(value)
        else:
            bad["kv_param"][at, 0, side, :, pos % 16, k % 2] = float(value)
        o = torch.full_like(clean, 9.0)
        call(o, q, **bad, layer_idx=0, seqlen_indptr=starts, window=window, sinks=sinks)
        sees = pos <= place
        if window:
            sees &= (place - pos < window) | (pos < sinks)
        assert torch.equal(o[~sees], clean[~sees]), k
        if side == 1 and f16:
            assert not bool(torch.isfinite(o[sees][:, :, dims]).any()) and torch.equal(o[sees][:, :, ~dims], clean[sees][:, :, ~dims]), k
        elif side == 1 or value == "nan":
            assert not bool(torch.isfinite(o[sees]).any()), k


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("heads,group,window,sinks", [(2, 2, 0, 0), (2, 2, 40, 3), (1, 8, 0, 0)])
@pytest.mark.parametrize("news", [[1], [30], [300]])
def test_few_rows_that_see_a_key_which_is_no_number(news, heads, group, window, sinks, f16):
    """They are not finite, and the others are as if it were any other (the kernel of 16 and of 32 rows)."""
    lens = [400]
    specs, q, starts = make(50 + news[0], 16, lens, news, heads, group, f16, layers=1)
    call = kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4
    clean = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    call(clean, q, **specs, layer_idx=0, seqlen_indptr=starts, window=window, sinks=sinks)
    place = torch.arange(400 - news[0], 400, device=DEV)
    for k, pos in enumerate((399, 395, 380, 150, 1)):
        bad = {**specs, "kv_data": specs["kv_data"].clone(), "kv_param": specs["kv_param"].clone()}
        at = int(specs["kv_indices"][pos // 16])
        if f16:
            bad["kv_data"][at, 0, 0, :, pos % 16, 7] = float("nan")
        else:
            bad["kv_param"][at, 0, 0, :, pos % 16, k % 2] = float("nan")
        o = torch.full_like(clean, 9.0)
        call(o, q, **bad, layer_idx=0, seqlen_indptr=starts, window=window, sinks=sinks)
        sees = pos <= place
        if window:
            sees &= (place - pos < window) | (pos < sinks)
        assert torch.equal(o[~sees], clean[~sees]) and not bool(torch.isfinite(o[sees]).any()), k


@pytest.mark.parametrize("f16", [False, True])
def test_a_call_twice_gives_the_same_bits(f16):
    for lens, news, heads, group in (([700], [256], 28, 8), ([4513], [512], 32, 1)):
        specs, q, starts = make(15, 16, lens, news, heads, group, f16, layers=1)
        first, second = (torch.empty(q.shape, dtype=torch.float16, device=DEV) for _ in range(2))
        for o in (first, second):
            (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **specs, layer_idx=0, seqlen_indptr=starts, max_new_len=news[0], max_seq_len=lens[0])
        assert torch.equal(first, second)


@pytest.mark.parametrize("f16", [False, True])
def test_pages_beyond_32_bit_offsets(f16):
    """A pool of more than 2^32 bytes, its last pages in use: the same bits as from a small one."""
    lens, news = [600, 90], [250, 6]
    specs, q, starts = make(5, 16, lens, news, 28, 8, f16, layers=2, spare=0)
    per, data = specs["kv_data"].shape[0], specs["kv_data"]
    total = (5 << 30) // (data[0].numel() * data.element_size())
    pool = {name: torch.empty((total, *specs[name].shape[1:]), dtype=specs[name].dtype, device=DEV) for name in ("kv_data", "kv_param")}
    for name, t in pool.items():
        t[total - per:] = specs[name]
    assert pool["kv_data"].numel() * data.element_size() > 1 << 32
    outs = [torch.empty_like(q) for _ in range(2)]
    for o, used in zip(outs, (specs, {**specs, **pool, "kv_indices": specs["kv_indices"] + (total - per)})):
        (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **used, layer_idx=1, seqlen_indptr=starts)
    assert torch.equal(*outs)

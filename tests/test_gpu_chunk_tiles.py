"""Attention of new tokens over the paged cache at sizes that go to the kernel of 256 rows (some 57000 rows and more in a call: 224 tiles of 256 rows are one turn
of the chip, 1792 of 32 would be several), against the definition in 64 bits and with the tolerances of test_gpu_chunk.py."""
import gc

import pytest
import torch

from quarot_amd import _lib
from tests.test_gpu_chunk import check, make, scale_values

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

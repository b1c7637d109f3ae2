"""One shared prefix whose tiles of 256 rows are dealt out in shares (csrc/qr_deal.h; test_prefix_shares.py goes through its arithmetic), against the 64-bit definition and with
the tolerances of test_gpu_shared.py, in workspaces of arbitrary contents of which nothing behind the asked-for bytes is touched."""
import gc

import pytest
import torch

from quarot_amd import _lib
from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV
from tests.test_gpu_shared import check_lse, definition, make_shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_goes_back():
    """What the module's tests allocated goes back to the device behind them (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def check_hints(f16, page_size, prefix_len, lens, news, heads, group, hints):
    step = max(news) == 1
    specs, prefix, q, starts = make_shared(prefix_len + heads, page_size, [prefix_len], None, lens, news, heads, group, f16)
    (want, tol), (lse_want, lse_tol) = definition(specs, prefix, q, [prefix_len], None, lens, news, 1)
    call = kv.batch_shared_f16 if f16 else kv.batch_shared_i4
    for hint in hints:
        counted = hint or prefix["prefix_indices"].numel() * page_size             # (the room of the page list where there is no hint)
        need = _lib.lib().qr_batch_shared_workspace_bytes(int(f16), q.shape[0], heads * group, heads, len(lens), max(news), max(lens), 0, 0, 1, counted)
        outs = []
        for fill in (255, 0, 60):                          # NaN; states of sum 0; finite numbers
            ws = torch.full((need + 65536,), fill, dtype=torch.uint8, device=DEV)
            o, lse = torch.full(q.shape, float("nan"), dtype=torch.float16, device=DEV), torch.full(q.shape[:2], float("nan"), device=DEV)
            call(o, q, **specs, layer_idx=1, **prefix, seqlen_indptr=None if step else starts, max_new_len=max(news), max_seq_len=max(lens), max_prefix_len=hint, lse=lse,
                 workspace=ws)
            assert bool((ws[need:] == fill).all()), (hint, fill)
            off = (o.double() - want).abs()
            assert bool((off <= tol).all()), f"hint {hint}, {fill}: {float((off / tol.clamp(min=1e-30)).nan_to_num(nan=float('inf')).max())} of what is allowed"
            check_lse(lse, lse_want, lse_tol)
            outs.append(o)
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]), hint


@pytest.mark.parametrize("prefix_len,tokens,heads,group", [(10000, 32, 8, 8), (10176, 31, 8, 8), (10048, 64, 4, 8), (10000, 128, 1, 16)])
def test_31_shares_and_a_fraction_to_a_tile(prefix_len, tokens, heads, group):
    """Fp16 pages, eight tiles: 251 to 254 shares of five steps would touch 33 states of a tile."""
    check_hints(True, 16, prefix_len, [1 + i % 5 for i in range(tokens)], [1] * tokens, heads, group, [prefix_len, 0])


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("page_size,prefix_len,hints,tokens,new,heads,group", [
    (16, 1000, [16384, 1 << 40], 32, 1, 8, 8), (16, 640, [8000, 100000], 64, 1, 8, 8), (7, 70, [1500, 20000], 300, 1, 1, 2), (64, 129, [30000], 20, 40, 2, 8),
    (128, 64, [16384], 40, 1, 8, 8), (16, 1, [5000], 40, 1, 8, 8)])
def test_prefixes_far_shorter_than_their_hint(page_size, prefix_len, hints, tokens, new, heads, group, f16):
    """Fewer steps than the launch has workgroups: a tile's states have no gaps, which the workspace's contents would fill."""
    check_hints(f16, page_size, prefix_len, [new + i % 5 for i in range(tokens)], [new] * tokens, heads, group, [*hints, prefix_len, 0])


@pytest.mark.parametrize("f16", [False, True])
def test_a_page_list_with_room_for_more(f16):
    """Without a hint the launch is cut for what the page list has room for, here eight times the prefix."""
    prefix_len, lens, news = 700, [3] * 40, [1] * 40
    specs, prefix, q, _ = make_shared(4, 16, [prefix_len], None, lens, news, 8, 8, f16)
    (want, tol), _ = definition(specs, prefix, q, [prefix_len], None, lens, news, 1)
    more = {**prefix, "prefix_indices": torch.cat([prefix["prefix_indices"], prefix["prefix_indices"][:1].repeat(8 * 44)])}
    o = torch.empty(q.shape, dtype=torch.float16, device=DEV)
    (kv.batch_shared_f16 if f16 else kv.batch_shared_i4)(o, q, **specs, layer_idx=1, **more, workspace=torch.full((1 << 28,), 255, dtype=torch.uint8, device=DEV))
    assert bool(((o.double() - want).abs() <= tol).all())

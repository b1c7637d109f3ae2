"""Attention of new tokens whose bounds count more than q has rows for, as build_page_tables gives them for `tokens` fewer than the new ones: the rows that there are keep the
positions that the tables and the append kernels give them."""
import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, definition, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("lens,news,heads,group,tokens,window,sinks,hint", [
    ([50, 90, 10], [20, 60, 5], 2, 2, 50, 0, 0, 0), ([50, 90], [20, 60], 2, 2, 21, 0, 0, 0), ([50, 90], [2, 30], 2, 2, 5, 20, 3, 0), ([900], [12], 1, 2, 3, 0, 0, 900),
    ([500, 700], [100, 256], 28, 8, 300, 0, 0, 0), ([500, 700], [100, 256], 28, 8, 300, 33, 2, 0), ([4513], [600], 32, 1, 512, 0, 0, 4513)])
def test_new_tokens_behind_the_last_row_are_left_out(lens, news, heads, group, tokens, window, sinks, hint, f16):
    specs, q, starts = make(60 + tokens, 16, lens, news, heads, group, f16, layers=1)
    want, tol = (t[:tokens] for t in definition(specs, q, lens, news, 0, window, sinks))
    some = q[:tokens].contiguous()
    o = torch.full_like(some, float("nan"))
    (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, some, **specs, layer_idx=0, seqlen_indptr=starts, max_seq_len=hint, window=window, sinks=sinks)
    assert bool(((o.double() - want).abs() <= tol).all())


def test_tables_append_and_attention_with_fewer_tokens_than_are_new():
    """build_page_tables, quantize_append_kv_i4 and batch_chunk_i4 on 20 of 26 new tokens: those 20 are stored and attend as with all 26, where no later one is seen."""
    lens, news, heads, tokens = [40, 33], [14, 12], 2, 20
    lengths, fresh = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in (lens, news))
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = (torch.randn(sum(news), heads, 128, generator=g, device=DEV).half() for _ in range(3))
    outs, pools = [], []
    for n in (sum(news), tokens):
        t = kv.build_page_tables(lengths, 16, 3, new_lengths=fresh, tokens=n)
        pool = {"kv_data": torch.full((6, 1, 2, heads, 16, 64), 17, dtype=torch.uint8, device=DEV), "kv_param": torch.full((6, 1, 2, heads, 16, 2), 0.5, dtype=torch.float16, device=DEV)}
        specs = {**pool, **{name: t[name] for name in ("kv_indptr", "kv_indices", "last_page_offset")}}
        kv.quantize_append_kv_i4(**specs, k=k[:n].contiguous(), v=v[:n].contiguous(), seqlen_indptr=t["seqlen_indptr"], layer_idx=0)
        outs.append(torch.empty(n, heads, 128, dtype=torch.float16, device=DEV))
        kv.batch_chunk_i4(outs[-1], q[:n].contiguous(), **specs, layer_idx=0, seqlen_indptr=t["seqlen_indptr"])
        pools.append(pool["kv_data"].permute(0, 4, 1, 2, 3, 5).reshape(96, 2, heads, 64)[t["slots"][:tokens]])
    assert torch.equal(*pools) and torch.equal(outs[0][:tokens], outs[1])

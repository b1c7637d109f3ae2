"""Attention of new tokens and page tables: calls whose sizes nothing could be computed for come back as errors, on the native route and on the one in Python."""
import pytest
import torch

from quarot_amd import _lib
from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, make

pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["native", "python"])
def route(request, monkeypatch):
    if not request.param:
        monkeypatch.setattr(_lib.host, "chunk", lambda *a: None)
        monkeypatch.setattr(_lib.host, "build_page_tables", lambda *a: None)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("axis,match", [(3, "multiple"), (4, "invalid size"), (0, "invalid size"), (1, "layer_idx")])
def test_caches_without_heads_entries_pages_or_layers(axis, match, f16, route):
    specs, q, starts = make(1, 16, [20, 5], [3, 2], 2, 2, f16)
    empty = {**specs, **{name: specs[name].narrow(axis, 0, 0).contiguous() for name in ("kv_data", "kv_param")}}
    with pytest.raises(RuntimeError, match=match):
        (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(torch.empty_like(q), q, **empty, layer_idx=0, seqlen_indptr=starts)


def test_new_tokens_that_32_bits_do_not_count(route):
    n = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    for tokens in (1 << 30, 1 << 31, 1 << 45):
        with pytest.raises(RuntimeError, match="below 2.30"):
            kv.build_page_tables(n, 16, 2, new_lengths=n, tokens=tokens)

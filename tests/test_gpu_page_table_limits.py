"""build_page_tables at its limits."""
import gc

import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_page_tables import DEV, by_hand

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    """What a test allocated goes back to the device behind it (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def test_new_tokens_of_more_than_31_bits_together():
    """Their bounds stay at 2^31 - 1, behind every token that there is, instead of turning negative."""
    lengths, new = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([3, 40, 5], [2, (1 << 31) - 1, 7]))
    got = kv.build_page_tables(lengths, 16, 3, new_lengths=new, tokens=4)
    assert got["seqlen_indptr"].tolist() == [0, 2, (1 << 31) - 1, (1 << 31) - 1]
    assert got["positions"].tolist() == [1, 2, 40 - ((1 << 31) - 1), 41 - ((1 << 31) - 1)] and got["slots"].tolist() == [1, 2, -1, -1]
    assert got["kv_indptr"].tolist() == [0, 1, 4, 5]


@pytest.mark.parametrize("batch", [2047, 2048, 2049, 4096, 5000])
def test_several_sequences_to_a_workgroup(batch):
    lengths, new = [(37 * b) % 50 for b in range(batch)], [(11 * b) % 5 - 1 for b in range(batch)]
    table = torch.randint(-1, 1 << 20, (batch, 5), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    tokens = sum(max(n, 0) for n in new)
    for asked, rows in ((tokens + 900, table), (tokens - 900, None)):
        got = kv.build_page_tables(*(torch.tensor(lengths, dtype=torch.int32, device=DEV), 16, 5), block_table=None if rows is None else rows.to(DEV),
                                   new_lengths=torch.tensor(new, dtype=torch.int32, device=DEV), tokens=asked)
        want = by_hand(lengths, 16, 5, None if rows is None else rows.tolist(), new, asked)
        for name, w in zip(("kv_indptr", "kv_indices", "last_page_offset", "seqlen_indptr", "positions", "slots"), want):
            assert got[name].tolist() == w, name


def test_more_sequences_than_a_launch_has_workgroups():
    """2^24 and some of no, one and two tokens on one page each."""
    batch = (1 << 24) + 777
    lengths = (torch.arange(batch, device=DEV) % 3).int()
    got = kv.build_page_tables(lengths, 2, 1, new_lengths=lengths, tokens=int(lengths.sum()) + 5)
    held = lengths > 0
    start = lambda v: torch.nn.functional.pad(v.cumsum(0), (1, 0))
    assert torch.equal(got["kv_indptr"], start(held.int()).int()) and torch.equal(got["last_page_offset"], lengths)
    assert torch.equal(got["seqlen_indptr"], start(lengths).int())
    pages, of = torch.nonzero(held)[:, 0], torch.repeat_interleave(torch.arange(batch, device=DEV), lengths.long())
    assert torch.equal(got["kv_indices"][:pages.numel()], pages.int()) and bool((got["kv_indices"][pages.numel():] == -1).all())
    at = torch.arange(of.numel(), device=DEV) - start(lengths)[of]
    assert torch.equal(got["positions"][:-5], at) and torch.equal(got["slots"][:-5], 2 * of + at)
    assert got["positions"][-5:].tolist() == got["slots"][-5:].tolist() == [-1] * 5

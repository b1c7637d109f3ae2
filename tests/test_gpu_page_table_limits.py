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

"""Attention of new tokens over the paged cache: what wrong or missing hints may cost, without a GPU (the workspace function plans as the call does)."""
import ctypes

import pytest

from quarot_amd import _lib

STATE = 132 * 4                                            # bytes of a row's partial state


@pytest.fixture(scope="module")
def size():
    return _lib.lib().qr_batch_chunk_workspace_bytes


@pytest.mark.parametrize("fp16", [0, 1])
@pytest.mark.parametrize("tokens", [17, 4096, 100000, 1 << 20])
def test_a_hint_below_what_some_sequence_must_have_counts_as_that(size, fp16, tokens):
    """One sequence has all tokens whatever the hint says, one of three a third of them."""
    for hint in (1, 2, 16, tokens - 1):
        assert size(fp16, tokens, 64, 8, 1, hint, 30000, 0, 0) == size(fp16, tokens, 64, 8, 1, tokens, 30000, 0, 0)
    third = -(-tokens // 3)
    assert size(fp16, tokens, 64, 8, 3, 1, 30000, 0, 0) == size(fp16, tokens, 64, 8, 3, third, 30000, 0, 0)


@pytest.mark.parametrize("fp16", [0, 1])
def test_partial_states_have_a_bound(size, fp16):
    """1 GiB, whatever the hints; whole states of every row."""
    for tokens in (1, 16, 100, 513, 3000, 20000, 100000, 1 << 20, 1 << 23):
        for heads, kv_heads in ((64, 8), (32, 32), (8, 1), (1, 1)):
            for batch in (1, 3, 16, 200, 100000):
                for hint in (0, 1, 7, 400, tokens):
                    for length in (0, 100, 5000, 1 << 20, (1 << 63) - 1):
                        for window, sinks in ((0, 0), (1000, 4)):
                            need = size(fp16, tokens, heads, kv_heads, batch, hint, length, window, sinks)
                            assert need <= 1 << 30 and need % (tokens * heads * STATE) == 0, (tokens, heads, batch, hint, length, window)


def test_no_workspace_for_what_the_call_refuses(size):
    assert size(0, 1 << 27, 8, 2, 3, 1, 4096, 0, 0) == 0   # tokens times heads
    assert size(0, 5, 2050, 2, 1, 5, 4096, 0, 0) == 0      # query heads to a key head
    assert size(0, 5, 8, 2, 1 << 31, 5, 4096, 0, 0) == 0
    assert size(0, (1 << 62) + 1, 8, 2, 3, 1, 4096, 0, 0) == 0


def test_lengths_windows_and_sinks_of_63_bits_count_as_longer_than_any_sequence(size):
    huge = (1 << 63) - 1
    for tokens in (1, 5, 600):
        long = size(0, tokens, 32, 32, 1, tokens, 1 << 30, 0, 0)
        for window, sinks in ((0, 0), (huge, 0), (huge, huge), (huge - 70, 3), (1, huge)):
            assert size(0, tokens, 32, 32, 1, tokens, huge, window, sinks) == long


@pytest.mark.parametrize("entry", ["qr_batch_chunk_i4", "qr_batch_chunk_f16"])
def test_key_heads_that_no_launch_holds_are_refused(size, entry):
    at = ctypes.c_void_p(4096)                             # never dereferenced
    heads = 65537
    assert getattr(_lib.lib(), entry)(at, heads * 128, at, heads * 128, 0, None, 1, heads, at, at, at, at, at, 1, 1, 0, heads, 16, 128, 1, 0, 0, 0, 0, None, 0, None) == -2
    assert size(0, 1, heads, heads, 1, 1, 4096, 0, 0) == 0

"""Page tables at the C entry point, without a GPU: counts that 32 bits do not hold are refused before any launch."""
import ctypes

import pytest

from quarot_amd import _lib


@pytest.mark.parametrize("tokens", [1 << 30, (1 << 31) - 1, 1 << 31, 1 << 40])
def test_new_tokens_that_32_bits_do_not_count(tokens):
    """(the kernel's loop over a sequence's new tokens would step past 2^31 - 1 and write in front of the slots)"""
    at = ctypes.c_void_p(4096)                             # never dereferenced
    assert _lib.lib().qr_build_page_tables(at, at, 3, 16, 4, at, 4, tokens, at, at, at, at, at, at, None) == -2

"""Attention of new tokens and page tables at the C entry points, without a GPU: wrong arguments come back as codes before any launch, workspaces
are sized without one."""
import ctypes

import pytest

from quarot_amd import _lib

NULL, SHAPE, ALIGN, DTYPE = -1, -2, -4, -5


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def _chunk_args(**changes):
    at = ctypes.c_void_p(4096)          # never dereferenced
    args = dict(o=at, o_stride=1024, q=at, q_stride=1024, had=0, starts=at, tokens=5, q_heads=8, data=at, param=at, indptr=at, indices=at, last=at, pages=10,
                layers=2, layer=1, heads=2, page_size=16, head_dim=128, batch=3, new=0, seq=0, window=0, sinks=0, workspace=None, bytes=0, stream=None)
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


@pytest.mark.parametrize("entry", ["qr_batch_chunk_i4", "qr_batch_chunk_f16"])
@pytest.mark.parametrize("code,change", [
    (NULL, {"o": None}), (NULL, {"q": None}), (NULL, {"data": None}), (NULL, {"indptr": None}), (NULL, {"indices": None}), (NULL, {"last": None}),
    (DTYPE, {"had": 2}), (DTYPE, {"had": -1}), (SHAPE, {"tokens": -1}), (SHAPE, {"q_heads": 7}), (SHAPE, {"q_heads": 0}), (SHAPE, {"window": -1}), (SHAPE, {"sinks": -1}),
    (SHAPE, {"new": -1}), (SHAPE, {"seq": -1}), (SHAPE, {"starts": None}), (SHAPE, {"q_stride": 1016}), (SHAPE, {"o_stride": 0}), (SHAPE, {"layer": 2}), (SHAPE, {"layer": -1}),
    (SHAPE, {"page_size": 0}), (SHAPE, {"heads": 0}), (SHAPE, {"batch": -1}), (SHAPE, {"tokens": 1 << 27}), (SHAPE, {"q_heads": 2050, "q_stride": 1 << 20, "o_stride": 1 << 20}),
    (ALIGN, {"q": ctypes.c_void_p(4104)}), (ALIGN, {"o": ctypes.c_void_p(4098)}), (ALIGN, {"q_stride": 1028}), (ALIGN, {"o_stride": 1026})])
def test_chunk_argument_errors(lib, entry, code, change):
    assert getattr(lib, entry)(*_chunk_args(**change)) == code


@pytest.mark.parametrize("entry", ["qr_batch_chunk_i4", "qr_batch_chunk_f16"])
def test_chunk_of_nothing(lib, entry):
    assert getattr(lib, entry)(*_chunk_args(tokens=0)) == 0
    assert getattr(lib, entry)(*_chunk_args(batch=0)) == 0


def test_chunk_workspace_needs_no_gpu(lib):
    size = lib.qr_batch_chunk_workspace_bytes
    for fp16 in (0, 1):
        assert size(fp16, 5, 32, 32, 1, 5, 0, 0, 0) == 0                       # no length: not split
        assert size(fp16, 0, 32, 32, 1, 0, 4096, 0, 0) == 0
        assert size(fp16, 5, 31, 32, 1, 5, 4096, 0, 0) == 0                    # (the call itself refuses it)
        one = size(fp16, 5, 32, 32, 1, 5, 4096, 0, 0)
        assert one > 0 and one % (5 * 32 * 132 * 4) == 0                       # whole states of every row
        assert size(fp16, 5, 32, 32, 1, 5, 1 << 20, 100, 4) <= one             # a window's positions count, not the sequence's
        for tokens in (1, 7, 33, 100, 513, 5000):
            for length in (1, 100, 4097, 1 << 20):
                need = size(fp16, tokens, 64, 8, 3, tokens, length, 0, 0)
                assert need % (tokens * 64 * 132 * 4) == 0 and need // (tokens * 64 * 132 * 4) in {0, *range(2, 33)}


def _table_args(**changes):
    at = ctypes.c_void_p(4096)
    args = dict(lengths=at, news=at, batch=3, page_size=16, max_pages=4, table=at, stride=4, tokens=5, indptr=at, indices=at, last=at, starts=at, positions=at, slots=at,
                stream=None)
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


@pytest.mark.parametrize("code,change", [
    (NULL, {"lengths": None}), (NULL, {"indptr": None}), (NULL, {"indices": None}), (NULL, {"last": None}), (NULL, {"starts": None}), (NULL, {"positions": None}),
    (NULL, {"slots": None}), (SHAPE, {"page_size": 0}), (SHAPE, {"max_pages": 0}), (SHAPE, {"batch": -1}), (SHAPE, {"stride": 3}), (SHAPE, {"tokens": -1}),
    (SHAPE, {"news": None}), (SHAPE, {"max_pages": 1 << 40, "stride": 1 << 40}), (SHAPE, {"batch": 1 << 29, "max_pages": 1 << 10, "stride": 1 << 10})])
def test_table_argument_errors(lib, code, change):
    assert lib.qr_build_page_tables(*_table_args(**change)) == code


def test_tables_of_nothing(lib):
    assert lib.qr_build_page_tables(*_table_args(batch=0)) == 0


def test_chunk_workspace_of_absurd_lengths(lib):
    """Nothing overflows: lengths, windows and sinks of 63 bits only size the launch."""
    huge = (1 << 63) - 1
    usual = lib.qr_batch_chunk_workspace_bytes(0, 5, 32, 32, 1, 5, 4096, 0, 0)
    for window, sinks in ((huge, 0), (5, huge), (huge, huge)):
        assert lib.qr_batch_chunk_workspace_bytes(0, 5, 32, 32, 1, 5, 4096, window, sinks) == usual
    assert lib.qr_batch_chunk_workspace_bytes(0, 5, 32, 32, 1, 5, huge >> 1, 0, 0) >= usual

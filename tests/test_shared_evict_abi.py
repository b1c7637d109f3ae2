"""Shared prefixes and eviction at the C entry points, without a GPU: wrong arguments come back as codes before any launch, workspaces are sized without one."""
import ctypes

import pytest

from quarot_amd import _lib

NULL, SHAPE, UNSUPPORTED, ALIGN, DTYPE, WORKSPACE = -1, -2, -3, -4, -5, -6
AT = ctypes.c_void_p(4096)              # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _lib.lib()


def changed(args, changes):
    assert set(changes) <= set(args)
    return list({**args, **changes}.values())


def shared_args(**changes):
    return changed(dict(o=AT, o_stride=1024, lse=AT, q=AT, q_stride=1024, had=0, starts=AT, tokens=5, q_heads=8, data=AT, param=AT, indptr=AT, indices=AT, last=AT, pages=10,
                        layers=2, layer=1, heads=2, page_size=16, head_dim=128, batch=3, new=0, seq=0, window=0, sinks=0, p_indptr=AT, p_indices=AT, p_last=AT, members=None,
                        prefixes=1, prefix=0, workspace=None, bytes=0, stream=None), changes)


@pytest.mark.parametrize("entry", ["qr_batch_shared_i4", "qr_batch_shared_f16"])
@pytest.mark.parametrize("code,change", [
    (NULL, {"o": None}), (NULL, {"q": None}), (NULL, {"data": None}), (NULL, {"indptr": None}), (NULL, {"p_indptr": None}), (NULL, {"p_indices": None}), (NULL, {"p_last": None}),
    (DTYPE, {"had": 2}), (SHAPE, {"tokens": -1}), (SHAPE, {"q_heads": 7}), (SHAPE, {"window": -1}), (SHAPE, {"window": 5}), (SHAPE, {"new": -1}), (SHAPE, {"prefix": -1}),
    (SHAPE, {"prefixes": -1}), (SHAPE, {"prefixes": 2}), (SHAPE, {"prefixes": 1 << 31, "members": AT}), (SHAPE, {"starts": None}), (SHAPE, {"q_stride": 1016}), (SHAPE, {"layer": 2}),
    (SHAPE, {"tokens": 1 << 27}), (SHAPE, {"tokens": 1 << 25}), (ALIGN, {"q": ctypes.c_void_p(4104)}), (ALIGN, {"o_stride": 1026}), (ALIGN, {"lse": ctypes.c_void_p(4098)}), (WORKSPACE, {}),
    (WORKSPACE, {"workspace": ctypes.c_void_p(4104), "bytes": 1 << 30}), (WORKSPACE, {"workspace": AT, "bytes": 1000})])
def test_shared_argument_errors(lib, entry, code, change):
    assert getattr(lib, entry)(*shared_args(**change)) == code


@pytest.mark.parametrize("entry", ["qr_batch_shared_i4", "qr_batch_shared_f16"])
def test_shared_of_nothing(lib, entry):
    assert getattr(lib, entry)(*shared_args(tokens=0)) == 0
    assert getattr(lib, entry)(*shared_args(batch=0)) == 0


def test_shared_workspace_needs_no_gpu(lib):
    size = lib.qr_batch_shared_workspace_bytes
    for fp16 in (0, 1):
        assert size(fp16, 0, 32, 32, 1, 0, 4096, 0, 0, 1, 0) == 0
        assert size(fp16, 5, 31, 32, 1, 5, 4096, 0, 0, 1, 0) == 0
        assert size(fp16, 5, 32, 32, 5, 1, 0, 0, 0, 0, 0) == 0                  # no prefix, not split: nothing to join
        assert size(fp16, 5, 32, 32, 1, 5, 4096, 0, 0, 0, 0) == lib.qr_batch_chunk_workspace_bytes(fp16, 5, 32, 32, 1, 5, 4096, 0, 0)
        for tokens in (1, 7, 33, 513, 5000):
            for length in (0, 1, 4097, 1 << 20, (1 << 62)):
                for prefixes in (1, 3):
                    need = size(fp16, tokens, 64, 8, 3, tokens, 100, 0, 0, prefixes, length)
                    states, rest = divmod(need, tokens * 64 * 132 * 4)
                    assert rest == 0 and 1 <= states <= 64


def weights_args(**changes):
    return changed(dict(weights=AT, capacity=100, q=AT, q_stride=1024, had=0, lse=AT, starts=AT, tokens=5, q_heads=8, data=AT, param=AT, indptr=AT, indices=AT, last=AT, pages=10,
                        layers=2, layer=1, heads=2, page_size=16, head_dim=128, batch=3, new=0, seq=0, window=0, sinks=0, workspace=None, bytes=0, stream=None), changes)


@pytest.mark.parametrize("entry", ["qr_accumulate_weights_i4", "qr_accumulate_weights_f16"])
@pytest.mark.parametrize("code,change", [
    (NULL, {"weights": None}), (NULL, {"q": None}), (NULL, {"lse": None}), (NULL, {"data": None}), (NULL, {"last": None}), (DTYPE, {"had": 3}), (SHAPE, {"capacity": -1}),
    (SHAPE, {"tokens": -1}), (SHAPE, {"q_heads": 7}), (SHAPE, {"window": -1}), (SHAPE, {"sinks": -1}), (SHAPE, {"seq": -1}), (SHAPE, {"starts": None}), (SHAPE, {"q_stride": 1016}),
    (SHAPE, {"layer": 2}), (SHAPE, {"tokens": 1 << 27}), (SHAPE, {"q_heads": 2050, "q_stride": 1 << 20}), (ALIGN, {"q": ctypes.c_void_p(4104)}), (ALIGN, {"q_stride": 1028}),
    (ALIGN, {"weights": ctypes.c_void_p(4098)}), (ALIGN, {"lse": ctypes.c_void_p(4097)})])
def test_weights_argument_errors(lib, entry, code, change):
    assert getattr(lib, entry)(*weights_args(**change)) == code


@pytest.mark.parametrize("entry", ["qr_accumulate_weights_i4", "qr_accumulate_weights_f16"])
def test_weights_of_nothing(lib, entry):
    for change in ({"tokens": 0}, {"batch": 0}, {"capacity": 0}):
        assert getattr(lib, entry)(*weights_args(**change)) == 0


def heavy_args(**changes):
    return changed(dict(weights=AT, capacity=100, lengths=AT, batch=3, heads=2, keep=50, sinks=4, recent=10, kept=AT, left=AT, stream=None), changes)


@pytest.mark.parametrize("code,change", [
    (NULL, {"weights": None}), (NULL, {"lengths": None}), (NULL, {"kept": None}), (NULL, {"left": None}), (SHAPE, {"batch": -1}), (SHAPE, {"heads": 0}), (SHAPE, {"capacity": -1}),
    (SHAPE, {"capacity": 1 << 40}), (SHAPE, {"keep": -1}), (SHAPE, {"keep": 1 << 40}), (SHAPE, {"sinks": -1}), (SHAPE, {"recent": -1}), (SHAPE, {"sinks": 41}), (SHAPE, {"recent": (1 << 63) - 1}),
    (SHAPE, {"batch": 1 << 22}), (SHAPE, {"batch": 1 << 21}), (ALIGN, {"weights": ctypes.c_void_p(4098)}), (ALIGN, {"kept": ctypes.c_void_p(4098)})])
def test_heavy_argument_errors(lib, code, change):
    assert lib.qr_heavy_positions(*heavy_args(**change)) == code


def keep_args(**changes):
    return changed(dict(kept=AT, keep=50, data=AT, param=AT, indptr=AT, indices=AT, last=AT, pages=10, layers=2, layer=1, heads=2, page_size=16, head_dim=128, batch=3, weights=AT,
                        capacity=100, stream=None), changes)


@pytest.mark.parametrize("entry", ["qr_keep_positions_i4", "qr_keep_positions_f16"])
@pytest.mark.parametrize("code,change", [
    (NULL, {"kept": None}), (NULL, {"data": None}), (NULL, {"param": None}), (NULL, {"indices": None}), (SHAPE, {"keep": -1}), (SHAPE, {"keep": 1 << 31}), (SHAPE, {"capacity": -1}),
    (SHAPE, {"layer": 2}), (SHAPE, {"batch": 1 << 20}), (SHAPE, {"batch": 1 << 30, "heads": 1 << 30}), (ALIGN, {"kept": ctypes.c_void_p(4098)}), (ALIGN, {"weights": ctypes.c_void_p(4098)})])
def test_keep_argument_errors(lib, entry, code, change):
    assert getattr(lib, entry)(*keep_args(**change)) == code


def test_nothing_stays_of_nothing(lib):
    assert lib.qr_heavy_positions(*heavy_args(batch=0)) == 0
    for entry in ("qr_keep_positions_i4", "qr_keep_positions_f16"):
        assert getattr(lib, entry)(*keep_args(batch=0)) == 0


def test_new_lengths_apart_from_the_lengths(lib):
    """A workgroup per key head reads a sequence's length, and one of them writes its new one."""
    assert lib.qr_heavy_positions(*heavy_args()) == UNSUPPORTED
    assert lib.qr_heavy_positions(*heavy_args(left=ctypes.c_void_p(AT.value + 8))) == UNSUPPORTED
    assert lib.qr_heavy_positions(*heavy_args(lengths=ctypes.c_void_p(AT.value + 8))) == UNSUPPORTED


@pytest.mark.parametrize("entry", ["qr_batch_shared_i4", "qr_batch_shared_f16"])
def test_rows_that_one_launch_joins(lib, entry):
    """16 rows take 256 threads of the launch that joins, which has fewer than 2^32."""
    many = dict(q_heads=1, heads=1, o_stride=128, q_stride=128)
    assert getattr(lib, entry)(*shared_args(tokens=(1 << 28) - 15, **many)) == SHAPE
    assert getattr(lib, entry)(*shared_args(tokens=(1 << 28) - 16, **many)) == WORKSPACE           # (none was given)

"""Attention of new tokens over the paged cache for batches whose workgroups do not fit one launch: more than 2^32 threads where the largest number of new tokens is not
given, and more sequences times heads than one launch has workgroups."""
import gc

import pytest
import torch

from quarot_amd.transformers import kv_cache as kv
from tests.test_gpu_chunk import DEV, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def memory_goes_back():
    """What a test allocated goes back to the device behind it (others fill the memory up to a limit)."""
    yield
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def cache_of(pages, heads, f16, seed):
    """A pool of pages of one position."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    if f16:
        data = torch.randn(pages, 1, 2, heads, 1, 128, generator=g, device=DEV, dtype=torch.float16)
        return data, torch.zeros(pages, 1, 2, heads, 1, 2, dtype=torch.float16, device=DEV), g
    data = torch.randint(0, 256, (pages, 1, 2, heads, 1, 64), generator=g, device=DEV, dtype=torch.uint8)
    param = torch.rand(pages, 1, 2, heads, 1, 2, generator=g, device=DEV, dtype=torch.float32)
    return data, (param * torch.tensor([0.5, 3.0], device=DEV) + 0.05).half(), g


def vectors(data, param, side):
    """fp64 [pages, heads, 128]; and what a vector's entries are made of: code times scale and zero point, in size."""
    if data.dtype == torch.float16:
        x = data[:, 0, side, :, 0].double()
        return x, x.abs()
    x, p = data[:, 0, side, :, 0], param[:, 0, side, :, 0].double()
    codes = torch.stack([x & 15, x >> 4], -1).flatten(-2).double() * p[..., :1]
    return codes - p[..., 1:], codes + p[..., 1:]


@pytest.mark.parametrize("f16", [False, True])
def test_many_sequences_without_hints(f16):
    """300000 sequences of no, one and two tokens, one key head; of a second token's two logits and values the result is known."""
    lens = torch.arange(300000, device=DEV) % 3
    start = torch.nn.functional.pad(lens.cumsum(0), (1, 0)).int()
    tokens = int(start[-1])
    data, param, g = cache_of(tokens, 1, f16, 1)
    q = torch.randn(tokens, 1, 128, generator=g, device=DEV).half()
    o = torch.full_like(q, float("nan"))
    specs = {"kv_data": data, "kv_param": param, "kv_indptr": start, "kv_indices": torch.arange(tokens, device=DEV, dtype=torch.int32), "last_page_offset": (lens > 0).int()}
    (kv.batch_chunk_f16 if f16 else kv.batch_chunk_i4)(o, q, **specs, layer_idx=0, seqlen_indptr=start)
    (keys, terms), (values, size) = ([t[:, 0] for t in vectors(data, param, side)] for side in (0, 1))
    second = torch.zeros(tokens, dtype=torch.bool, device=DEV)
    second[start[:-1][lens == 2].long() + 1] = True
    before = torch.arange(tokens, device=DEV) - second.long()
    q64 = q[:, 0].double()
    logits = [(q64 * k).sum(-1, keepdim=True) / 128 ** 0.5 for k in (keys, keys[before])]
    w = torch.where(second[:, None], torch.sigmoid(logits[0] - logits[1]), 1.0)
    want = w * values + (1 - w) * values[before]
    # test_gpu_chunk.py's tolerance: roundings of the output and of the weights, and twice the larger error of the two logits, of exp2's arguments and of the sums
    far = 2 * torch.maximum(*[140 * 2.0 ** -24 * (q64.abs() * t).sum(-1, keepdim=True) / 128 ** 0.5 + 2.0 ** -21 * t.sum(-1, keepdim=True) / 128 ** 0.5 for t in (terms, terms[before])])
    far += 2.0 ** -22 * (1 + 1.5 * torch.maximum(logits[0].abs(), logits[1].abs())) + 201 * 2.0 ** -24
    off = 2.0 ** -11 * (2 * want.abs() + w * values.abs() + (1 - w) * values[before].abs()) + 2.0 ** -25 * (values.abs() + values[before].abs() + 2 * want.abs() + 1)
    off += far * (w * size + (1 - w) * size[before])
    assert bool(((o[:, 0].double() - want).abs() <= off).all())


@pytest.mark.parametrize("f16", [False, True])
def test_a_ragged_batch_of_thousands_without_hints(f16):
    news = [28 + (b % 5 - 2) * (b % 7) for b in range(5000)]
    specs, q, starts = make(3, 16, news, news, 1, 1, f16, layers=1)
    assert 5000 * min(4096, sum(news) // 32) * 256 > 1 << 32
    check(specs, q, starts, news, news, layer=0, hints=(False,))


@pytest.mark.parametrize("bounds", [False, True])
def test_more_sequences_and_heads_than_a_launch_has_workgroups(bounds):
    """90000 sequences of one token, 64 heads, workgroups of 768 threads (the hint says that there is much to read): every output is its own value."""
    batch, heads = 90000, 64
    assert batch * heads * 768 > 1 << 32
    data, param, g = cache_of(batch, heads, False, 2)
    q = torch.randn(batch, heads, 128, generator=g, device=DEV, dtype=torch.float16)
    o = torch.full_like(q, float("nan"))
    each = torch.arange(batch + 1, device=DEV, dtype=torch.int32)
    kv.batch_chunk_i4(o, q, kv_data=data, kv_param=param, kv_indptr=each, kv_indices=each[:-1], last_page_offset=torch.ones_like(each[:-1]), layer_idx=0,
                      seqlen_indptr=each if bounds else None, max_new_len=1, max_seq_len=100000)
    for at in range(0, batch, 10000):
        want, size = vectors(data[at:at + 10000], param[at:at + 10000], 1)
        # (the only weight counts as rounded; sums of products of code and scale in 32 bits)
        assert bool(((o[at:at + 10000].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -18 * size).all())

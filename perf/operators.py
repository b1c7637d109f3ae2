"""Attention of new tokens over the paged KV cache, with and without a sliding window, and the page tables it goes by,
as measurable cases.

  chunk    several new tokens of every sequence against everything that its pages hold (their own keys included):
           a prompt that arrives in pieces, the second turn of a conversation, drafted tokens.
  window   the same where a token sees the last `window` positions and the first `sinks` ones; with new = 1 it is the
           step of one token per sequence.
  tables   page lists, offsets, positions and slots from the lengths of a batch's requests.

Head counts, widths and page sizes are those of the package's benchmark workloads (32 and 40 heads of 128, 64 query heads
on 8 key heads, pages of 16 to 128), lengths run from one token to a context of 32768.
"""
import math

import torch

own = False

HEAD_DIM = 128
LAYERS, LAYER = 2, 1                                       # the cache holds two layers, the second one is read


def _attention_case(name, kind, batch, new, cached, heads, kv_heads, pages="i4", page=16, ragged=False, fused=False, window=0, sinks=0):
    return {"name": name, "kind": kind, "batch": batch, "new": new, "cached": cached, "heads": heads, "kv_heads": kv_heads,
            "pages": pages, "page": page, "ragged": ragged, "fused": fused, "window": window, "sinks": sinks}


def listed():
    return [
        # five drafted tokens of one short conversation are verified: all latency
        _attention_case("chunk_5_after_203_32heads", "chunk", 1, 5, 203, 32, 32),
        # a serving batch in which every sequence brings a few tokens, lengths all different, queries a slice of a fused projection
        _attention_case("chunk_7x_to_37_after_2100_64on8", "chunk", 7, 37, 2100, 64, 8, ragged=True, fused=True),
        # a second turn: an ordinary question behind a conversation
        _attention_case("chunk_512_after_4001_32heads", "chunk", 1, 512, 4001, 32, 32),
        # prompts that arrive in one piece, grouped heads, unequal lengths
        _attention_case("chunk_8x_to_2048_64on8", "chunk", 8, 2048, 0, 64, 8, ragged=True),
        # a long document, its last piece of 2048 tokens: the largest
        _attention_case("chunk_2048_after_30720_64on8", "chunk", 1, 2048, 30720, 64, 8, page=64),
        # the cache that keeps its vectors in fp16, odd sizes
        _attention_case("chunk_f16_3x777_after_1500_40heads", "chunk", 3, 777, 1500, 40, 40, pages="f16"),
        # one conversation far beyond its window: one token
        _attention_case("window_step_1x30001_32heads", "window", 1, 1, 30000, 32, 32, window=1024, sinks=4),
        # a full serving batch with grouped heads: one token each
        _attention_case("window_step_32x4001_64on8", "window", 32, 1, 4000, 64, 8, window=2048, sinks=4),
        # the same step on fp16 pages
        _attention_case("window_step_f16_16x2500_40heads", "window", 16, 1, 2499, 40, 40, pages="f16", window=1000, sinks=16),
        # a piece of a long prompt through a window
        _attention_case("window_2x1501_after_8000_32heads", "window", 2, 1501, 8000, 32, 32, window=1024, sinks=4),
        # page tables of three sequences at a step
        {"name": "tables_3x500", "kind": "tables", "batch": 3, "length": 500, "new": 1, "page": 16, "table": False},
        # and of a large batch of mixed work, pages from an allocator
        {"name": "tables_256x8192_new512", "kind": "tables", "batch": 256, "length": 8192, "new": 512, "page": 16, "table": True},
    ]


_MOST_SCORES = 64 * 2048 * 32768                          # rows x positions of the largest listed case
_MOST_POSITIONS = 32 * 4096 * 8                           # positions x key heads of the cache


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["chunk"] * 5 + ["window"] * 4 + ["tables"] * 2)
    if kind == "tables":
        length = _log(rng, 1, 16384)
        return {"kind": kind, "batch": _log(rng, 1, 512), "length": length, "new": _log(rng, 1, min(length, 512)),
                "page": rng.choice([16, 16, 32, 64, 128, 5]), "table": rng.random() < 0.6}
    while True:
        heads, kv_heads = rng.choice([(32, 32), (40, 40), (64, 8), (64, 8), (32, 8), (12, 4), (8, 1)])
        step = kind == "window" and rng.random() < 0.5
        case = _attention_case("", kind, _log(rng, 1, 48), 1 if step else _log(rng, 1, 4096), rng.choice([0, 1, 1, 1]) * _log(rng, 1, 30720),
                               heads, kv_heads, rng.choice(["i4", "i4", "i4", "f16"]), rng.choice([16, 16, 32, 64, 128, 7]),
                               rng.random() < 0.5, rng.random() < 0.3, _log(rng, 16, 8192) if kind == "window" else 0,
                               rng.choice([0, 1, 4, 16, 100]) if kind == "window" else 0)
        del case["name"]
        most = case["new"] + case["cached"]
        if case["batch"] * heads * case["new"] * most <= _MOST_SCORES and case["batch"] * kv_heads * most <= _MOST_POSITIONS:
            return case


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence; a ragged batch has those with most new tokens hold least."""
    n, new, cached = case["batch"], case["new"], case["cached"]
    if not case["ragged"]:
        return [new] * n, [new + cached] * n
    news = [max(1, new * (n - i) // n) for i in range(n)]
    return news, [a + cached * (i + 1) // n for i, a in enumerate(news)]


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _vectors(gen, *shape):
    """Keys or values: N(0, 1), one in two hundred fifteen times as large."""
    x = _randn(gen, *shape)
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.005, x * 15, x)


def _quantised(x):
    """fp16 vectors -> packed 4-bit codes and {scale, zero}: scale = max(max - min, 1e-5) / 15, zero = -min, low nibble first."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, zero = ((high - low).clamp(min=1e-5) / 15).half(), (-low).half()
    codes = torch.round((x + zero.float()) / scale.float()).clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, torch.cat([scale, zero], dim=-1)


def _start(lengths):
    return torch.nn.functional.pad(torch.cumsum(lengths, 0, dtype=torch.int32), (1, 0))


def _prepare_attention(case, gen):
    news, lens = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in _lengths(case))
    heads, kv_heads, page, tokens = case["heads"], case["kv_heads"], case["page"], sum(_lengths(case)[0])
    per = [(n + page - 1) // page for n in _lengths(case)[1]]
    total = sum(per)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    shape = (total, LAYERS, 2, kv_heads, page)
    if case["pages"] == "i4":
        kv_data = torch.zeros(*shape, HEAD_DIM // 2, dtype=torch.uint8, device="cuda")
        kv_param = torch.zeros(*shape, 2, dtype=torch.float16, device="cuda")
        for side in (0, 1):
            kv_data[:, LAYER, side], kv_param[:, LAYER, side] = _quantised(_vectors(gen, total, kv_heads, page, HEAD_DIM).half().float())
    else:
        kv_data = torch.zeros(*shape, HEAD_DIM, dtype=torch.float16, device="cuda")
        kv_param = torch.tensor([1.0, 0.0], dtype=torch.float16, device="cuda").repeat(*shape, 1)
        for side in (0, 1):
            kv_data[:, LAYER, side] = _vectors(gen, total, kv_heads, page, HEAD_DIM).half()
    width = heads * HEAD_DIM
    q = _randn(gen, tokens, width + (2 * kv_heads * HEAD_DIM if case["fused"] else 0)).half()[:, :width].view(tokens, heads, HEAD_DIM)
    return {"case": case, "q": q, "seqlens": None if case["new"] == 1 else _start(news), "max_new": max(_lengths(case)[0]),
            "max_len": max(_lengths(case)[1]), "specs": {
                "kv_data": kv_data, "kv_param": kv_param, "kv_indptr": _start((lens + page - 1) // page), "kv_indices": order,
                "last_page_offset": (lens - 1) % page + 1}}


def _tables_lengths(case):
    n = case["batch"]
    lens = [max(1, case["length"] - case["length"] * i // (2 * n)) for i in range(n)]
    return lens, [max(1, min(a, case["new"] * (i + 1) // n)) for i, a in enumerate(lens)]


def _prepare_tables(case, gen):
    lens, news = _tables_lengths(case)
    page, n = case["page"], case["batch"]
    most = (max(lens) + page - 1) // page
    # the requests come in an order of their own
    at = torch.randperm(n, generator=gen, device="cuda")
    table = torch.randperm(n * most, generator=gen, device="cuda").to(torch.int32).view(n, most) if case["table"] else None
    as_tensor = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")[at].contiguous()
    return {"case": case, "lengths": as_tensor(lens), "new_lengths": as_tensor(news), "tokens": sum(news), "max_pages": most, "table": table}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return _prepare_tables(case, gen) if case["kind"] == "tables" else _prepare_attention(case, gen)


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_vectors(specs, most):
    """The cached vectors of all sequences, padded to `most` pages: fp32 [2, batch, key heads, positions, 128]."""
    first, end = specs["kv_indptr"][:-1].long(), specs["kv_indptr"][1:].long()
    at = first[:, None] + torch.arange(most, device="cuda")
    at = torch.minimum(at, (end - 1).clamp(min=0)[:, None])
    pages = specs["kv_indices"].long()[at]
    data = specs["kv_data"][pages, LAYER]                 # [batch, pages, 2, key heads, page, bytes or halves]
    if data.dtype == torch.uint8:
        param = specs["kv_param"][pages, LAYER].float()
        data = torch.stack([data & 15, data >> 4], dim=-1).flatten(-2).float() * param[..., :1] - param[..., 1:]
    data = data.float().permute(2, 0, 3, 1, 4, 5)
    return data.reshape(*data.shape[:3], -1, HEAD_DIM)


def _plain_attention(state):
    case, specs, q = state["case"], state["specs"], state["q"]
    page, kv_heads, group = case["page"], case["kv_heads"], case["heads"] // case["kv_heads"]
    batch, most_new = case["batch"], state["max_new"]
    keys, values = _plain_vectors(specs, (state["max_len"] + page - 1) // page)
    seqlens = state["seqlens"] if state["seqlens"] is not None else torch.arange(batch + 1, device="cuda")
    seqlens = seqlens.long()
    lens = (specs["kv_indptr"].diff().long() - 1) * page + specs["last_page_offset"].long()
    token = torch.arange(q.shape[0], device="cuda")
    row = torch.arange(most_new, device="cuda")
    padded = q[(seqlens[:-1, None] + row).clamp(max=q.shape[0] - 1)].float()          # [batch, new, heads, 128]
    padded = padded.view(batch, most_new, kv_heads, group, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * most_new, HEAD_DIM)
    scores = torch.matmul(padded, keys.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(HEAD_DIM))
    scores = scores.view(batch, kv_heads, group, most_new, -1)
    place = (lens - seqlens.diff())[:, None, None] + row[:, None]                     # [batch, new, 1]
    position = torch.arange(scores.shape[-1], device="cuda")
    hidden = position > place
    if case["window"]:
        hidden |= (position <= place - case["window"]) & (position >= case["sinks"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(batch, kv_heads, group * most_new, -1), values).view(batch, kv_heads, group, most_new, HEAD_DIM) / total
    of = torch.searchsorted(seqlens[1:].contiguous(), token, right=True)
    return [out.permute(0, 3, 1, 2, 4)[of, token - seqlens[of]].reshape(q.shape).half()]


def _plain_tables(state):
    case, lens, news, page = state["case"], state["lengths"].long(), state["new_lengths"].long(), state["case"]["page"]
    batch, most = case["batch"], state["max_pages"]
    table = state["table"].long() if state["table"] is not None else (
        torch.arange(most, device="cuda") * batch + torch.arange(batch, device="cuda")[:, None])
    pages = (lens + page - 1) // page
    start = lambda n: torch.nn.functional.pad(torch.cumsum(n, 0), (1, 0))
    indptr, seqlens = start(pages), start(news)
    entry = torch.arange(batch * most, device="cuda")
    of = torch.searchsorted(indptr[1:].contiguous(), entry, right=True)
    known = of.clamp(max=batch - 1)
    indices = torch.where(of < batch, table[known, (entry - indptr[known]).clamp(0, most - 1)], -1)
    token = torch.arange(state["tokens"], device="cuda")
    of = torch.searchsorted(seqlens[1:].contiguous(), token, right=True)
    position = lens[of] - news[of] + token - seqlens[of]
    slot = table[of, position // page] * page + position % page
    return [indptr.int(), indices.int(), ((lens - 1) % page + 1).int(), seqlens.int(), position, slot]


# ---- the package's calls ---------------------------------------------------------------------------------------------

def _own_attention(state):
    from quarot_amd.transformers import kv_cache as kv
    case, q = state["case"], state["q"]
    o = torch.empty(q.shape, dtype=torch.float16, device=q.device)
    call = kv.batch_chunk_i4 if case["pages"] == "i4" else kv.batch_chunk_f16
    call(o, q, **state["specs"], layer_idx=LAYER, seqlen_indptr=state["seqlens"], max_new_len=state["max_new"], max_seq_len=state["max_len"],
         window=case["window"], sinks=case["sinks"])
    return [o]


def _own_tables(state):
    from quarot_amd.transformers import kv_cache as kv
    t = kv.build_page_tables(state["lengths"], state["case"]["page"], state["max_pages"], block_table=state["table"],
                             new_lengths=state["new_lengths"], tokens=state["tokens"])
    return [t[name] for name in ("kv_indptr", "kv_indices", "last_page_offset", "seqlen_indptr", "positions", "slots")]


def run(state):
    if own:
        return _own_tables(state) if state["case"]["kind"] == "tables" else _own_attention(state)
    return _plain_tables(state) if state["case"]["kind"] == "tables" else _plain_attention(state)


def _seen(case, place):
    """How many positions a token at position `place` sees."""
    if not case["window"] or place + 1 <= case["window"]:
        return place + 1
    return case["window"] + min(case["sinks"], place + 1 - case["window"])


def work(case):
    if case["kind"] == "tables":
        lens, news = _tables_lengths(case)
        pages = sum((n + case["page"] - 1) // case["page"] for n in lens)
        most = case["batch"] * ((max(lens) + case["page"] - 1) // case["page"])
        return {"bytes": 4 * (2 * case["batch"] + (pages if case["table"] else 0) + 3 * case["batch"] + 2 + most) + 16 * sum(news), "flops": 0}
    bytes_, pairs = 0, 0
    vector = 136 if case["pages"] == "i4" else 512          # a key and a value
    for new, length in zip(*_lengths(case)):
        first = length - new                                # the first new token's position
        read = length
        if case["window"]:
            read -= max(0, first - case["window"] + 1 - case["sinks"])
        bytes_ += read * case["kv_heads"] * vector + new * case["heads"] * 4 * HEAD_DIM
        pairs += sum(_seen(case, p) for p in range(first, length))
    return {"bytes": bytes_, "flops": 4.0 * HEAD_DIM * pairs * case["heads"]}


def exact(case, seed):
    """Each sequence and key head by itself, in 64 bits, from the definition."""
    if case["kind"] == "tables":
        return None
    state = prepare(case, seed)
    specs, page, group = state["specs"], case["page"], case["heads"] // case["kv_heads"]
    bounds, pages = specs["kv_indptr"].tolist(), specs["kv_indices"].long()
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    token = 0
    for b, (new, length) in enumerate(zip(*_lengths(case))):
        held = pages[bounds[b]:bounds[b + 1]]
        place = torch.arange(length - new, length, device="cuda").repeat(group)[:, None]
        j = torch.arange(length, device="cuda")[None]
        sees = j <= place
        if case["window"]:
            sees &= (place - j < case["window"]) | (j < case["sinks"])
        for h in range(case["kv_heads"]):
            sides = []
            for side in (0, 1):
                x = specs["kv_data"][held, LAYER, side, h].reshape(len(held) * page, -1)[:length]
                if case["pages"] == "i4":
                    p = specs["kv_param"][held, LAYER, side, h].reshape(len(held) * page, 2)[:length].double()
                    y = torch.empty(length, HEAD_DIM, dtype=torch.float64, device="cuda")
                    y[:, 0::2], y[:, 1::2] = torch.remainder(x, 16).double(), torch.div(x, 16, rounding_mode="floor").double()
                    x = y * p[:, 0:1] - p[:, 1:2]
                sides.append(x.double())
            queries = state["q"][token:token + new, h * group:(h + 1) * group].double().transpose(0, 1).reshape(group * new, HEAD_DIM)
            logits = queries @ sides[0].t() / math.sqrt(HEAD_DIM)
            weights = torch.softmax(torch.where(sees, logits, -math.inf), dim=-1)
            out[token:token + new, h * group:(h + 1) * group] = (weights @ sides[1]).view(group, new, HEAD_DIM).transpose(0, 1)
        token += new
    return [out]

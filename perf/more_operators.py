"""Attention with shared prefixes over the paged KV cache, and eviction from it by accumulated attention weight, as measurable cases.

  shared   new tokens of sequences that begin with the same text, whose pages are held once: one prefix of the whole batch, or
           several, each of some of its sequences.
  weights  what the new tokens' attention gives to every cached position, added to that position's sum.
  heavy    the positions that stay: the first ones, the last ones, and those of the largest sums between them.
  keep     their vectors, parameters and sums moved to the front of the sequence's pages.

Head counts, widths and page sizes are those of the package's benchmark workloads (32 and 40 heads of 128, 64 query heads
on 8 key heads, pages of 16 to 128), lengths run from one token to a context of 32768.
"""
import math

import torch

own = False

HEAD_DIM = 128
LAYERS, LAYER = 2, 1                                       # the cache holds two layers, the second one is worked on


def _shared_case(name, batch, prefixes, prefix, new, held, heads, kv_heads, pages="i4", page=16, ragged=False, fused=False):
    return {"name": name, "kind": "shared", "batch": batch, "prefixes": prefixes, "prefix": prefix, "new": new, "cached": held, "heads": heads, "kv_heads": kv_heads,
            "pages": pages, "page": page, "ragged": ragged, "fused": fused}


def _weights_case(name, batch, new, cached, heads, kv_heads, pages="i4", page=16, ragged=False, fused=False, window=0, sinks=0):
    return {"name": name, "kind": "weights", "batch": batch, "new": new, "cached": cached, "heads": heads, "kv_heads": kv_heads,
            "pages": pages, "page": page, "ragged": ragged, "fused": fused, "window": window, "sinks": sinks}


def _evict_case(name, kind, batch, length, keep, kv_heads, sinks, recent, pages="i4", page=16, ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "length": length, "keep": keep, "kv_heads": kv_heads, "sinks": sinks, "recent": recent,
            "pages": pages, "page": page, "ragged": ragged}


def listed():
    return [
        # four answers to one prompt, just begun: all latency
        _shared_case("shared_4_one_after_1200_32heads", 4, 1, 1200, 1, 100, 32, 32),
        # a serving batch behind one long system prompt, every answer of its own length, grouped heads
        _shared_case("shared_64_one_after_8192_64on8", 64, 1, 8192, 1, 700, 64, 8, ragged=True),
        # three prompts, each of a part of the batch, a few drafted tokens of every sequence, the cache that keeps its vectors in fp16
        _shared_case("shared_f16_3of30_to_5_after_2999_40heads", 30, 3, 2999, 5, 333, 40, 40, pages="f16", ragged=True, fused=True),
        # questions of some length about one document: the largest
        _shared_case("shared_16_to_256_after_16384_64on8", 16, 1, 16384, 256, 0, 64, 8, page=64, ragged=True),
        # one conversation, one token: all latency
        _weights_case("weights_step_1x3001_32heads", 1, 1, 3000, 32, 32),
        # a full serving batch with grouped heads, one token each
        _weights_case("weights_step_32x4001_64on8", 32, 1, 4000, 64, 8),
        # a few tokens of every sequence through a window, fp16 pages, queries a slice of a fused projection
        _weights_case("weights_f16_5x_to_37_after_1777_40heads", 5, 37, 1777, 40, 40, pages="f16", ragged=True, fused=True, window=1500, sinks=4),
        # the last piece of a long prompt: the largest
        _weights_case("weights_2048_after_14336_64on8", 1, 2048, 14336, 64, 8, page=64),
        # one conversation's heads are asked which positions stay
        _evict_case("heavy_1x2500_of_32heads", "heavy", 1, 2500, 1024, 32, 4, 256),
        # a full serving batch after its prompts
        _evict_case("heavy_32x_to_16384_of_8heads", "heavy", 32, 16384, 4096, 8, 4, 1024, ragged=True),
        # half of one conversation's cache goes
        _evict_case("keep_1024_of_2048_32heads", "keep", 1, 2048, 1024, 32, 4, 256),
        # and of a full serving batch's, on pages of fp16
        _evict_case("keep_f16_32x2000_of_8001_8heads", "keep", 32, 8001, 2000, 8, 4, 501, pages="f16", ragged=True),
    ]


_MOST_SHARED = 64 * 16 * 256 * 8192                        # rows x positions of the largest listed cases
_MOST_WEIGHTS = 64 * 2048 * 15360
_MOST_POSITIONS = 32 * 8001 * 8                            # positions x key heads of the cache
_MOST_KEPT = 32 * 2000 * 8                                 # and of what stays


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["shared"] * 4 + ["weights"] * 4 + ["heavy"] * 2 + ["keep"] * 2)
    while True:
        heads, kv_heads = rng.choice([(32, 32), (40, 40), (64, 8), (64, 8), (32, 8), (12, 4), (8, 1)])
        pages, page, ragged = rng.choice(["i4", "i4", "i4", "f16"]), rng.choice([16, 16, 32, 64, 128, 7]), rng.random() < 0.5
        if kind == "shared":
            batch = _log(rng, 1, 128)
            case = _shared_case("", batch, min(batch, rng.choice([1, 1, 1, 2, 3, 7])), _log(rng, 1, 30000), 1 if rng.random() < 0.5 else _log(rng, 1, 1024),
                                rng.choice([0, 1, 1]) * _log(rng, 1, 4096), heads, kv_heads, pages, page, ragged, rng.random() < 0.3)
            most, held = case["new"] + case["cached"], case["prefix"] * case["prefixes"]
            fits = batch * heads * case["new"] * (most + case["prefix"]) <= _MOST_SHARED and kv_heads * (batch * most + held) <= _MOST_POSITIONS
        elif kind == "weights":
            step = rng.random() < 0.5
            window = rng.choice([0, 0, 1]) * _log(rng, 16, 8192)
            case = _weights_case("", _log(rng, 1, 48), 1 if step else _log(rng, 1, 2048), rng.choice([0, 1, 1, 1]) * _log(rng, 1, 30000) or int(step), heads, kv_heads,
                                 pages, page, ragged, rng.random() < 0.3, window, rng.choice([0, 1, 4, 100]) if window else 0)
            most = case["new"] + case["cached"]
            fits = case["batch"] * heads * case["new"] * most <= _MOST_WEIGHTS and case["batch"] * kv_heads * most <= _MOST_POSITIONS
        else:
            length = _log(rng, 64, 32768)
            keep = _log(rng, 4, min(length * 3 // 4, 8192))
            sinks = min(keep // 2, rng.choice([0, 0, 1, 4, 100]))
            case = _evict_case("", kind, _log(rng, 1, 48), length, keep, kv_heads, sinks, int((keep - sinks) * rng.choice([0, 0.1, 0.25, 0.5, 0.75])), pages, page, ragged)
            fits = case["batch"] * kv_heads * length <= _MOST_POSITIONS and (kind == "heavy" or case["batch"] * kv_heads * min(keep, length) <= _MOST_KEPT)
        if fits:
            del case["name"]
            return case


def _lengths(case):
    """(new tokens, tokens of its own in the cache with them) of every sequence; a ragged batch has those with most new tokens hold least."""
    n, new, cached = case["batch"], case["new"], case["cached"]
    if not case["ragged"]:
        return [new] * n, [new + cached] * n
    news = [max(1, new * (n - i) // n) for i in range(n)]
    return news, [a + cached * (i + 1) // n for i, a in enumerate(news)]


def _prefixes(case):
    """(first sequence of every prefix and the end, positions of every prefix)"""
    n = case["prefixes"]
    return [case["batch"] * i // n for i in range(n + 1)], [max(1, case["prefix"] * (n - i) // n) for i in range(n)]


def _held(case):
    """Tokens of every sequence before an eviction."""
    n, length = case["batch"], case["length"]
    return [max(1, length - length * i // (2 * n)) for i in range(n)] if case["ragged"] else [length] * n


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _vectors(gen, *shape):
    """Keys or values: N(0, 1), one in two hundred fifteen times as large."""
    x = _randn(gen, *shape)
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.005, x * 15, x)


def _sums(gen, *shape):
    """Accumulated weights: spread over orders of magnitude as attention's are, one in twenty positions never attended to."""
    x = torch.exp(2 * _randn(gen, *shape) - 3)
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.05, 0, x)


def _quantised(x):
    """fp16 vectors -> packed 4-bit codes and {scale, zero}: scale = max(max - min, 1e-5) / 15, zero = -min, low nibble first."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale, zero = ((high - low).clamp(min=1e-5) / 15).half(), (-low).half()
    codes = torch.round((x + zero.float()) / scale.float()).clamp(0, 15).to(torch.uint8)
    return codes[..., 0::2] | codes[..., 1::2] << 4, torch.cat([scale, zero], dim=-1)


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _start(lengths):
    return torch.nn.functional.pad(torch.cumsum(lengths, 0, dtype=torch.int32), (1, 0))


def _pool(case, gen, total):
    kv_heads, page = case["kv_heads"], case["page"]
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
    return kv_data, kv_param


def _tables(lens, page, order):
    """Page tables of sequences that hold `lens` tokens, on the pages of `order` in turn."""
    lens = _int32(lens)
    return {"kv_indptr": _start((lens + page - 1) // page), "kv_indices": order, "last_page_offset": (lens - 1) % page + 1}


def _queries(case, gen, tokens):
    width = case["heads"] * HEAD_DIM
    wide = width + (2 * case["kv_heads"] * HEAD_DIM if case["fused"] else 0)
    return _randn(gen, tokens, wide).half()[:, :width].view(tokens, case["heads"], HEAD_DIM)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    page, kv_heads = case["page"], case["kv_heads"]
    state = {"case": case}
    lens = _lengths(case)[1] if case["kind"] in ("shared", "weights") else _held(case)
    if case["kind"] == "heavy":
        state["lengths"] = _int32(lens)
        place = torch.arange(max(lens), device="cuda")
        state["weights"] = torch.where(place < state["lengths"][:, None, None], _sums(gen, case["batch"], kv_heads, max(lens)), 0)
        return state
    count = sum((n + page - 1) // page for n in lens)
    shared = _prefixes(case)[1] if case["kind"] == "shared" else []
    total = count + sum((n + page - 1) // page for n in shared)
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    kv_data, kv_param = _pool(case, gen, total)
    state["specs"] = {"kv_data": kv_data, "kv_param": kv_param, **_tables(lens, page, order[:count].contiguous())}
    state["max_len"] = max(lens)
    if case["kind"] == "keep":
        # the sums go by a plain selection, as a program's own would
        weights = torch.where(torch.arange(max(lens), device="cuda") < _int32(lens)[:, None, None], _sums(gen, case["batch"], kv_heads, max(lens)), 0)
        state["weights"], state["kept"] = weights, _plain_heavy({"case": case, "lengths": _int32(lens), "weights": weights})[0]
        return state
    news = _lengths(case)[0]
    state["q"] = _queries(case, gen, sum(news))
    state["seqlens"] = None if case["new"] == 1 else _start(_int32(news))
    state["max_new"] = max(news)
    if case["kind"] == "shared":
        tables = _tables(shared, page, order[count:].contiguous())
        state["prefix"] = {"prefix_indptr": tables["kv_indptr"], "prefix_indices": tables["kv_indices"], "prefix_last_page_offset": tables["last_page_offset"],
                           "prefix_sequences": None if case["prefixes"] == 1 else _int32(_prefixes(case)[0])}
        state["max_prefix"] = max(shared)
        return state
    # the logarithms of the softmax's sums, which the attention has given, and sums of earlier steps
    state["lse"] = torch.empty(state["q"].shape[:2], dtype=torch.float32, device="cuda")
    token = 0
    bounds, pages = state["specs"]["kv_indptr"].tolist(), order.long()
    for b, (new, length) in enumerate(zip(news, lens)):
        for h in range(kv_heads):
            logits = _sequence_logits(state, pages[bounds[b]:bounds[b + 1]], h, token, new, length, torch.float32)
            of_rows = torch.logsumexp(logits, -1).view(new, -1)
            state["lse"][token:token + new, h * of_rows.shape[1]:(h + 1) * of_rows.shape[1]] = of_rows
        token += new
    place = torch.arange(max(lens), device="cuda")
    state["weights"] = torch.where(place < _int32([n - a for n, a in zip(lens, news)])[:, None, None], _sums(gen, case["batch"], kv_heads, max(lens)), 0)
    return state


def _sequence_side(state, held, side, h, length, dtype):
    """Keys (0) or values (1) of one key head on the pages `held`: [length, 128]."""
    specs, page = state["specs"], state["case"]["page"]
    x = specs["kv_data"][held, LAYER, side, h].reshape(len(held) * page, -1)[:length]
    if state["case"]["pages"] != "i4":
        return x.to(dtype)
    p = specs["kv_param"][held, LAYER, side, h].reshape(len(held) * page, 2)[:length].to(dtype)
    y = torch.empty(length, HEAD_DIM, dtype=dtype, device="cuda")
    y[:, 0::2], y[:, 1::2] = torch.remainder(x, 16).to(dtype), torch.div(x, 16, rounding_mode="floor").to(dtype)
    return y * p[:, 0:1] - p[:, 1:2]


def _sees(case, place, j):
    sees = j <= place
    if case.get("window"):
        sees &= (place - j < case["window"]) | (j < case["sinks"])
    return sees


def _sequence_logits(state, held, h, token, new, length, dtype):
    """Logits of the new tokens' rows (token by token, its query heads of key head h) against the sequence's positions."""
    case, group = state["case"], state["case"]["heads"] // state["case"]["kv_heads"]
    queries = state["q"][token:token + new, h * group:(h + 1) * group].to(dtype).reshape(new * group, HEAD_DIM)
    logits = queries @ _sequence_side(state, held, 0, h, length, dtype).t() / math.sqrt(HEAD_DIM)
    place = torch.arange(length - new, length, device="cuda").repeat_interleave(group)[:, None]
    return torch.where(_sees(case, place, torch.arange(length, device="cuda")[None]), logits, -math.inf)


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _plain_vectors(specs, indptr, indices, most, sides):
    """The cached vectors of all page lists, padded to `most` pages: fp32 [sides, lists, key heads, positions, 128]."""
    first, end = indptr[:-1].long(), indptr[1:].long()
    at = first[:, None] + torch.arange(most, device="cuda")
    at = torch.minimum(at, (end - 1).clamp(min=0)[:, None])
    pages = indices.long()[at]
    data = specs["kv_data"][pages, LAYER, :sides]         # [lists, pages, sides, key heads, page, bytes or halves]
    if data.dtype == torch.uint8:
        param = specs["kv_param"][pages, LAYER, :sides].float()
        data = torch.stack([data & 15, data >> 4], dim=-1).flatten(-2).float() * param[..., :1] - param[..., 1:]
    data = data.float().permute(2, 0, 3, 1, 4, 5)
    return data.reshape(*data.shape[:3], -1, HEAD_DIM)


def _plain_rows(state, seqlens, most_new):
    """The queries padded to `most_new` tokens a sequence: fp32 [batch, key heads, group * most_new, 128]; group outside."""
    case, q = state["case"], state["q"]
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    padded = q[(seqlens[:-1, None] + torch.arange(most_new, device="cuda")).clamp(max=q.shape[0] - 1)].float()
    return padded.view(case["batch"], most_new, kv_heads, group, HEAD_DIM).permute(0, 2, 3, 1, 4).reshape(case["batch"], kv_heads, group * most_new, HEAD_DIM)


def _plain_bounds(state):
    """Bounds of the new tokens, and how many tokens every sequence holds."""
    case, specs = state["case"], state["specs"]
    seqlens = (state["seqlens"] if state["seqlens"] is not None else torch.arange(case["batch"] + 1, device="cuda")).long()
    lens = (specs["kv_indptr"].diff().long() - 1) * case["page"] + specs["last_page_offset"].long()
    return seqlens, lens


def _plain_logits(state, seqlens, lens, keys):
    case = state["case"]
    batch, kv_heads, group, most_new = case["batch"], case["kv_heads"], case["heads"] // case["kv_heads"], state["max_new"]
    scores = torch.matmul(_plain_rows(state, seqlens, most_new), keys.transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(HEAD_DIM))
    scores = scores.view(batch, kv_heads, group, most_new, -1)
    place = (lens - seqlens.diff())[:, None, None] + torch.arange(most_new, device="cuda")[:, None]
    hidden = ~_sees(case, place, torch.arange(scores.shape[-1], device="cuda"))
    return scores.masked_fill_(hidden[:, None, None], -math.inf)


def _of_tokens(state, seqlens, padded):
    """[batch, key heads, group, new, ...] -> [tokens, heads, ...]"""
    token = torch.arange(state["q"].shape[0], device="cuda")
    of = torch.searchsorted(seqlens[1:].contiguous(), token, right=True)
    picked = padded.transpose(2, 3).transpose(1, 2)[of, token - seqlens[of]]
    return picked.reshape(*state["q"].shape[:2], *picked.shape[3:])


def _plain_shared(state):
    case, specs, page = state["case"], state["specs"], state["case"]["page"]
    kv_heads, group, most_new = case["kv_heads"], case["heads"] // case["kv_heads"], state["max_new"]
    seqlens, lens = _plain_bounds(state)
    keys, values = _plain_vectors(specs, specs["kv_indptr"], specs["kv_indices"], (state["max_len"] + page - 1) // page, 2)
    scores = _plain_logits(state, seqlens, lens, keys)                                # [batch, key heads, group, new, positions]
    most = scores.amax(-1, keepdim=True)
    scores.sub_(most).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(case["batch"], kv_heads, group * most_new, -1), values).view(case["batch"], kv_heads, group, most_new, HEAD_DIM)
    del scores, keys, values
    # each prefix by itself, with the rows of all tokens that it belongs to
    most, total, out = (_of_tokens(state, seqlens, t) for t in (most, total, out))
    prefix = state["prefix"]
    keys, values = _plain_vectors(specs, prefix["prefix_indptr"], prefix["prefix_indices"], (state["max_prefix"] + page - 1) // page, 2)
    held = (prefix["prefix_indptr"].diff().long() - 1) * page + prefix["prefix_last_page_offset"].long()
    sequences, lengths = _prefixes(case)
    first_tokens = [sum(_lengths(case)[0][:n]) for n in sequences]
    result = torch.empty(state["q"].shape, dtype=torch.float16, device="cuda")
    for i, length in enumerate(lengths):
        rows = slice(first_tokens[i], first_tokens[i + 1])
        q = state["q"][rows].float().view(-1, kv_heads, group, HEAD_DIM).transpose(0, 1).reshape(kv_heads, -1, HEAD_DIM)
        scores = torch.matmul(q, keys[i, :, :length].transpose(-1, -2).contiguous()).mul_(1 / math.sqrt(HEAD_DIM))
        scores.masked_fill_(torch.arange(length, device="cuda") >= held[i], -math.inf)
        own_most = most[rows].view(-1, kv_heads, group).transpose(0, 1).reshape(kv_heads, -1, 1)
        high = torch.maximum(scores.amax(-1, keepdim=True), own_most)
        scores.sub_(high).exp_()
        keep = torch.exp(own_most - high)
        by_head = lambda t: t[rows].view(-1, kv_heads, group, t.shape[-1]).transpose(0, 1).reshape(kv_heads, -1, t.shape[-1])
        both = (torch.matmul(scores, values[i, :, :length]) + by_head(out) * keep) / (scores.sum(-1, keepdim=True) + by_head(total) * keep)
        result[rows] = both.view(kv_heads, -1, group, HEAD_DIM).transpose(0, 1).reshape(-1, case["heads"], HEAD_DIM).half()
    return [result]


def _plain_weights(state):
    case, specs, page = state["case"], state["specs"], state["case"]["page"]
    seqlens, lens = _plain_bounds(state)
    keys = _plain_vectors(specs, specs["kv_indptr"], specs["kv_indices"], (state["max_len"] + page - 1) // page, 1)[0]
    scores = _plain_logits(state, seqlens, lens, keys)
    kv_heads, group, most_new = case["kv_heads"], case["heads"] // case["kv_heads"], state["max_new"]
    row = torch.arange(most_new, device="cuda")
    lse = state["lse"][(seqlens[:-1, None] + row).clamp(max=state["q"].shape[0] - 1)].view(case["batch"], most_new, kv_heads, group).permute(0, 2, 3, 1)
    there = (row < seqlens.diff()[:, None])[:, None, None]
    lse = torch.where(there, lse, math.inf)                                            # (rows that only fill up)
    added = scores.sub_(lse[..., None]).exp_().sum((2, 3), dtype=torch.float64)
    weights = state["weights"]
    weights.copy_(weights.double() + added[..., :weights.shape[-1]])
    return [weights]


def _plain_heavy(state):
    case, weights, lens = state["case"], state["weights"], state["lengths"].long()
    keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
    place = torch.arange(weights.shape[-1], device="cuda")
    length = lens[:, None, None]
    always = (place < sinks) | (place >= length - recent)
    rank = torch.where(always, math.inf, weights.double())
    rank = torch.where(place < length, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices              # ties: the lowest position first
    order = order[..., :keep]
    count = torch.clamp(lens, max=keep)[:, None, None]
    order = torch.where(torch.arange(order.shape[-1], device="cuda") < count, order, weights.shape[-1])
    kept = torch.full((*weights.shape[:2], keep), -1, dtype=torch.int32, device="cuda")
    order = torch.sort(order, dim=-1).values
    kept[..., :order.shape[-1]] = torch.where(order < weights.shape[-1], order, -1)
    return [kept, count.flatten().int()]


def _plain_keep(state):
    case, specs, kept, page = state["case"], state["specs"], state["kept"].long(), state["case"]["page"]
    first, weights = specs["kv_indptr"][:-1].long(), state["weights"]
    b, h, i = torch.nonzero(kept >= 0, as_tuple=True)
    source = kept[b, h, i]
    pages, entries = specs["kv_indices"].long()[first[b] + source // page], source % page
    to_pages, to_entries = specs["kv_indices"].long()[first[b] + i // page], i % page
    for t in (specs["kv_data"], specs["kv_param"]):
        for side in (0, 1):
            t[to_pages, LAYER, side, h, to_entries] = t[pages, LAYER, side, h, entries]
    moved = torch.where(kept >= 0, torch.gather(weights, -1, kept.clamp(min=0)), 0)
    weights.zero_()
    count = min(kept.shape[-1], weights.shape[-1])
    weights[..., :count] = moved[..., :count]
    return [specs["kv_data"], specs["kv_param"], weights]


# ---- the package's calls ---------------------------------------------------------------------------------------------

def _own_shared(state):
    from quarot_amd.transformers import kv_cache as kv
    case, q = state["case"], state["q"]
    o = torch.empty(q.shape, dtype=torch.float16, device=q.device)
    call = kv.batch_shared_i4 if case["pages"] == "i4" else kv.batch_shared_f16
    call(o, q, **state["specs"], layer_idx=LAYER, **state["prefix"], seqlen_indptr=state["seqlens"], max_new_len=state["max_new"], max_seq_len=state["max_len"],
         max_prefix_len=state["max_prefix"])
    return [o]


def _own_weights(state):
    from quarot_amd.transformers import kv_cache as kv
    case = state["case"]
    call = kv.accumulate_weights_i4 if case["pages"] == "i4" else kv.accumulate_weights_f16
    call(state["weights"], state["q"], state["lse"], **state["specs"], layer_idx=LAYER, seqlen_indptr=state["seqlens"], max_new_len=state["max_new"],
         max_seq_len=state["max_len"], window=case["window"], sinks=case["sinks"])
    return [state["weights"]]


def _own_heavy(state):
    from quarot_amd.transformers import kv_cache as kv
    case = state["case"]
    return list(kv.heavy_positions(state["weights"], state["lengths"], case["keep"], sinks=case["sinks"], recent=case["recent"]))


def _own_keep(state):
    from quarot_amd.transformers import kv_cache as kv
    call = kv.keep_positions_i4 if state["case"]["pages"] == "i4" else kv.keep_positions_f16
    call(state["kept"], **state["specs"], layer_idx=LAYER, weights=state["weights"])
    return [state["specs"]["kv_data"], state["specs"]["kv_param"], state["weights"]]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"shared": _own_shared, "weights": _own_weights, "heavy": _own_heavy, "keep": _own_keep}[kind](state)
    return {"shared": _plain_shared, "weights": _plain_weights, "heavy": _plain_heavy, "keep": _plain_keep}[kind](state)


def _seen(case, place):
    """How many positions a token at position `place` sees."""
    if not case.get("window") or place + 1 <= case["window"]:
        return place + 1
    return case["window"] + min(case["sinks"], place + 1 - case["window"])


def work(case):
    kind = case["kind"]
    if kind in ("heavy", "keep"):
        lens, heads = _held(case), case["kv_heads"]
        stay = sum(min(n, case["keep"]) for n in lens) * heads
        if kind == "heavy":
            return {"bytes": 4 * (sum(lens) * heads + case["batch"] * heads * case["keep"] + 2 * case["batch"]), "flops": 0}
        # (what moves: the kept entries of sequences that are longer; their sums, and the zeros behind them)
        moved = sum(case["keep"] - min(case["sinks"], case["keep"]) for n in lens if n > case["keep"]) * heads
        return {"bytes": 2 * moved * ((136 if case["pages"] == "i4" else 520) + 4) + 4 * stay + 4 * max(0, sum(lens) * heads - stay), "flops": 0}
    bytes_, pairs = 0, 0
    side = {"i4": 68, "f16": 256}[case["pages"]]
    sides = 2 if kind == "shared" else 1
    for new, length in zip(*_lengths(case)):
        first = length - new                                # the first new token's position
        read = length
        if case.get("window"):
            read -= max(0, first - case["window"] + 1 - case["sinks"])
        # q and o, or q, the sums' logarithms and the weights that are seen, read and written
        bytes_ += read * case["kv_heads"] * side * sides + new * case["heads"] * (4 * HEAD_DIM if kind == "shared" else 2 * HEAD_DIM + 4)
        bytes_ += 0 if kind == "shared" else read * case["kv_heads"] * 8
        pairs += sum(_seen(case, p) for p in range(first, length))
    if kind == "shared":
        sequences, lengths = _prefixes(case)
        news = _lengths(case)[0]
        for i, length in enumerate(lengths):
            bytes_ += length * case["kv_heads"] * side * 2
            pairs += length * sum(news[sequences[i]:sequences[i + 1]])
    return {"bytes": bytes_, "flops": 2.0 * sides * HEAD_DIM * pairs * case["heads"]}


# ---- from the definitions, in 64 bits --------------------------------------------------------------------------------

def _exact_attention(case, state):
    specs = state["specs"]
    kv_heads, group = case["kv_heads"], case["heads"] // case["kv_heads"]
    bounds, pages = specs["kv_indptr"].tolist(), specs["kv_indices"].long()
    shared = case["kind"] == "shared"
    if shared:
        prefix = state["prefix"]
        prefix_bounds, prefix_pages = prefix["prefix_indptr"].tolist(), prefix["prefix_indices"].long()
        sequences, lengths = _prefixes(case)
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda") if shared else state["weights"].double()
    for h in range(kv_heads):
        token, read = 0, -1
        for b, (new, length) in enumerate(zip(*_lengths(case))):
            held = pages[bounds[b]:bounds[b + 1]]
            logits = _sequence_logits(state, held, h, token, new, length, torch.float64)
            if shared:
                of = max(i for i, n in enumerate(sequences[:-1]) if n <= b)
                if of != read:
                    at, read = prefix_pages[prefix_bounds[of]:prefix_bounds[of + 1]], of
                    keys, values = (_sequence_side(state, at, side, h, lengths[of], torch.float64) for side in (0, 1))
                queries = state["q"][token:token + new, h * group:(h + 1) * group].double().reshape(new * group, HEAD_DIM)
                weights = torch.softmax(torch.cat([queries @ keys.t() / math.sqrt(HEAD_DIM), logits], -1), -1)
                o = weights @ torch.cat([values, _sequence_side(state, held, 1, h, length, torch.float64)])
                out[token:token + new, h * group:(h + 1) * group] = o.view(new, group, HEAD_DIM)
            else:
                lse = state["lse"][token:token + new, h * group:(h + 1) * group].double().reshape(new * group, 1)
                out[b, h, :length] += torch.exp(logits - lse).sum(0)
            token += new
    return [out]


def _exact_keep(case, state):
    specs, page = state["specs"], case["page"]
    bounds, pages, kept = specs["kv_indptr"].tolist(), specs["kv_indices"].long(), state["kept"]
    before, after = (specs["kv_data"], specs["kv_param"]), (specs["kv_data"].clone(), specs["kv_param"].clone())
    weights = torch.zeros_like(state["weights"])
    for b in range(case["batch"]):
        held = pages[bounds[b]:bounds[b + 1]]
        for h in range(case["kv_heads"]):
            stay = kept[b, h][kept[b, h] >= 0].long()
            for old, new in zip(before, after):
                for side in (0, 1):
                    rows = old[held, LAYER, side, h].flatten(0, 1)
                    rows[:len(stay)] = rows[stay]
                    new[held, LAYER, side, h] = rows.view(len(held), page, -1)
            weights[b, h, :len(stay)] = state["weights"][b, h, stay]
    return [None if case["pages"] == "i4" else after[0].double(), after[1].double(), weights.double()]


def exact(case, seed):
    if case["kind"] == "heavy":
        return None
    state = prepare(case, seed)
    return _exact_keep(case, state) if case["kind"] == "keep" else _exact_attention(case, state)

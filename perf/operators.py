"""Timed cases of the paged 8-bit KV cache operators and of the rotary embedding in front of them.

Four operators, as a decoder layer uses them between its QKV projection and its output projection:

``rotary``     rotary positions with several axes (time, height, width) on the query and key heads
``write``      new keys and values quantised into the pages of an E4M3 cache, one power-of-two
               (UE8M0) scale per block of 32 tokens and head
``read``       tokens of the cache back as 16-bit rows
``attention``  grouped-query attention of new tokens over that cache: one token per sequence
               (decode), a few (speculative verification), or a chunk of a prompt (prefill)

``run`` computes the plain form (elementary torch operations in 32 bits) or, with ``own`` set, makes
the package's calls.  ``exact`` computes the definition in 64 bits.
"""

import math
import random

import numpy as np
import torch

own = False

BLOCK = 32        # tokens that share a scale
MAX_CODE = 448.0  # largest finite E4M3 value
FLOOR_CODE = 28   # smallest scale the quantiser writes: 2^-99

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------- cases


def _attention(name, batch, context, query, q_heads, kv_heads, dim, page, dtype, ragged, causal=True):
    return {"name": name, "op": "attention", "batch": batch, "context": context, "query": query,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype,
            "ragged": ragged, "causal": causal}


def _cache_case(name, op, batch, context, query, kv_heads, dim, page, dtype, ragged):
    return {"name": name, "op": op, "batch": batch, "context": context, "query": query,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "ragged": ragged}


def _rotary(name, tokens, q_heads, kv_heads, dim, rotary_dim, axes, far, interleaved, dtype):
    return {"name": name, "op": "rotary", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "rotary_dim": rotary_dim, "axes": axes, "far": far,
            "interleaved": interleaved, "dtype": dtype}


def listed():
    return [
        # One user's first tokens after a short prompt: latency of a decode step's attention.
        _attention("decode_1x200", 1, 200, 1, 24, 4, 256, 32, "bf16", False),
        # One user deep in a long document: the whole GPU has to share one sequence.
        _attention("decode_1x131072", 1, 131072, 1, 24, 4, 256, 64, "bf16", False),
        # A serving batch of the 27B-class decoder, contexts of every length up to 8192.
        _attention("decode_32x8192_ragged", 32, 8192, 1, 24, 4, 256, 64, "bf16", True),
        # Speculative verification: up to four drafted tokens per sequence, narrower heads, f16.
        _attention("verify_48x4096_ragged", 48, 4096, 4, 32, 8, 128, 32, "f16", True),
        # Prefill of one whole prompt.
        _attention("prefill_1x8192", 1, 8192, 8192, 24, 4, 256, 128, "bf16", False),
        # Chunked prefill: ragged chunks of several prompts over contexts already in the cache.
        _attention("chunk_5x12000_ragged", 5, 12000, 1500, 16, 2, 128, 64, "bf16", True),
        # A decode batch appends one token to every sequence.
        _cache_case("write_32x1", "write", 32, 2048, 1, 4, 256, 64, "bf16", True),
        # A prompt's keys and values go into fresh pages.
        _cache_case("write_1x8191", "write", 1, 8191, 8191, 4, 256, 64, "bf16", False),
        # One short prompt back to 16 bits (prefix export, inspection).
        _cache_case("read_1x77", "read", 1, 77, 77, 8, 128, 32, "f16", False),
        # The cached contexts of a batch back to 16 bits.
        _cache_case("read_12x6000_ragged", "read", 12, 6000, 6000, 4, 256, 64, "bf16", True),
        # Decode batch with three position axes, a quarter of each head rotated.
        _rotary("rotary_17", 17, 24, 4, 256, 64, 3, 262144, True, "bf16"),
        # Prompt with image tokens: whole heads rotated, chunked sections.
        _rotary("rotary_8192", 8192, 32, 8, 128, 128, 3, 32768, False, "f16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "verify", "prefill", "write", "read", "rotary"])
    dtype = rng.choice(["bf16", "f16"])
    dim = rng.choice([64, 128, 256])
    page = rng.choice([32, 64, 128])
    kv = rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4])
    group = rng.choice([1, 2, 3, 4, 6, 8])
    ragged = rng.random() < 0.7
    if kind in ("decode", "verify"):
        batch = _log(rng, 1, 64)
        # as many cached tokens in all as the largest decode case at most
        context = _log(rng, 1, min(131072, (131072 * 4 * 256) // (batch * kv * dim)))
        query = 1 if kind == "decode" else min(rng.randint(2, 8), context)
        return _pure(_attention("", batch, context, query, kv * group, kv, dim, page, dtype, ragged))
    if kind == "prefill":
        batch = rng.randint(1, 4)
        query = _log(rng, 9, 4096 // batch)
        context = max(query, _log(rng, query, 8192))
        return _pure(_attention("", batch, context, query, kv * min(group, 4), kv, min(dim, 256), page,
                                dtype, ragged, rng.random() < 0.8))
    if kind in ("write", "read"):
        batch = _log(rng, 1, 64)
        context = _log(rng, 1, 8192 // batch * 4 if kind == "read" else 8192)
        query = context if kind == "read" else min(context, _log(rng, 1, max(1, 8192 // batch)))
        context = min(context, max(1, 131072 // batch))
        return _pure(_cache_case("", kind, batch, context, min(query, context), kv, dim, page, dtype,
                                 ragged))
    axes = rng.choice([1, 2, 3, 4])
    rotary_dim = rng.choice([dim, dim // 2, dim // 4])
    tokens = _log(rng, 1, 8192)
    return _pure(_rotary("", tokens, kv * group, kv, dim, rotary_dim, axes, _log(rng, 100, 1 << 20),
                         rng.random() < 0.5, dtype))


def _pure(case):
    return {key: value for key, value in case.items() if key != "name"}


def _lengths(case):
    """(cached length after the call, new tokens) of every sequence, from the case alone."""
    rng = random.Random(case["batch"] * 7919 + case["context"] * 31 + case["query"])
    lengths, news = [], []
    for index in range(case["batch"]):
        if case["ragged"] and index:
            length, new = rng.randint(1, case["context"]), rng.randint(1, case["query"])
        else:
            length, new = case["context"], case["query"]
        new = length if case["op"] == "read" else min(new, length)
        lengths.append(length)
        news.append(new)
    return lengths, news


# --------------------------------------------------------------------------- inputs


def _codes(shape, gen):
    """E4M3 codes of normally distributed values whose 4-sigma point is the largest code."""
    return (torch.randn(shape, device="cuda", generator=gen) * 112.0).clamp_(-MAX_CODE, MAX_CODE).to(
        torch.float8_e4m3fn).view(torch.uint8)


def _positions_of(lengths, news):
    """Host plan of the new tokens: sequence, position and index within the sequence of each row."""
    seq = np.repeat(np.arange(len(news)), news)
    index = np.concatenate([np.arange(n) for n in news]) if len(news) else np.zeros(0, np.int64)
    position = index + np.repeat(np.array(lengths) - np.array(news), news)
    return seq, position, index


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = torch.device("cuda")
    dtype = _DTYPES[case["dtype"]]
    if case["op"] == "rotary":
        tokens, dim, half = case["tokens"], case["dim"], case["rotary_dim"] // 2
        heads, axes = case["q_heads"] + case["kv_heads"], case["axes"]
        qk = torch.randn((tokens, heads * dim), device=dev, generator=gen).to(dtype)
        q = qk[:, : case["q_heads"] * dim].view(tokens, case["q_heads"], dim)
        k = qk[:, case["q_heads"] * dim :].view(tokens, case["kv_heads"], dim)
        positions = torch.randint(0, case["far"], (axes, tokens), device=dev, generator=gen)
        # sections: the first axis gets what an even split leaves over
        sections = [half // axes] * axes
        sections[0] += half - sum(sections)
        frequency = np.arange(half)
        if case["interleaved"]:
            axis = frequency % axes
            axis[frequency >= axes * np.array(sections)[axis]] = 0
        else:
            axis = np.repeat(np.arange(axes), sections)
        inv = 1.0e6 ** (-np.arange(half, dtype=np.float64) / half)
        return {"case": case, "q": q, "k": k, "positions": positions,
                "inv_freq": torch.from_numpy(inv).to(dev),
                "axis": torch.from_numpy(axis.astype(np.int32)).to(dev),
                "q_out": torch.empty((tokens, case["q_heads"], dim), dtype=dtype, device=dev),
                "k_out": torch.empty((tokens, case["kv_heads"], dim), dtype=dtype, device=dev)}

    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    lengths, news = _lengths(case)
    batch, total = case["batch"], sum(news)
    width = max(-(-n // page) for n in lengths)
    needed = sum(-(-n // page) for n in lengths)
    pages = needed + 3
    # pages of the pool in random order; entries behind a sequence's last page name no page
    order = torch.randperm(pages, device=dev, generator=gen).cpu().numpy()
    table = np.full((batch, width), -1, np.int32)
    at = 0
    for b, n in enumerate(lengths):
        count = -(-n // page)
        table[b, :count] = order[at : at + count]
        at += count
    shape = (pages, heads, page, dim)
    cache = {"k_values": _codes(shape, gen), "v_values": _codes(shape, gen)}
    for name in ("k_scales", "v_scales"):
        cache[name] = torch.randint(118, 122, (pages, heads, page // BLOCK), device=dev, generator=gen,
                                    dtype=torch.uint8)
    seq, position, index = _positions_of(lengths, news)
    state = {"case": case, **cache,
             "table": torch.from_numpy(table).to(dev),
             "lengths": torch.tensor(lengths, dtype=torch.int32, device=dev),
             "starts": None if case["op"] != "read" and case["query"] == 1 else torch.tensor(
                 np.concatenate([[0], np.cumsum(news)]), dtype=torch.int32, device=dev),
             "tokens": total, "widest": max(news), "longest": max(lengths),
             "seq": torch.from_numpy(seq).to(dev), "position": torch.from_numpy(position).to(dev),
             "index": torch.from_numpy(index).to(dev)}
    if case["op"] == "attention":
        # what lies behind a sequence's last token is whatever was there: any byte, NaN among them
        for b, n in enumerate(lengths):
            if n % page:
                last = int(table[b, n // page])
                for name in ("k_values", "v_values"):
                    tail = cache[name][last, :, n % page :]
                    tail.copy_(torch.randint(0, 256, tail.shape, device=dev, generator=gen,
                                             dtype=torch.uint8))
        q_heads = case["q_heads"]
        # the query heads are a slice of the projection's rows
        qkv = torch.randn((total, (q_heads + 2 * heads) * dim), device=dev, generator=gen)
        state["q"] = (2.0 * qkv).to(dtype)[:, : q_heads * dim].view(total, q_heads, dim)
        state["out"] = torch.empty((total, q_heads, dim), dtype=dtype, device=dev)
    elif case["op"] == "write":
        kv = torch.randn((total, 2 * heads * dim), device=dev, generator=gen)
        # keys have a few channels that are much larger than the others
        kv[:, :: max(1, dim // 4)] *= 8.0
        kv = kv.to(dtype)
        state["k"] = kv[:, : heads * dim].view(total, heads, dim)
        state["v"] = kv[:, heads * dim :].view(total, heads, dim)
        # (sequence, block) pairs that receive tokens, and each row's place in them
        pairs, first = [], []
        for b, (n, new) in enumerate(zip(lengths, news)):
            first.append(len(pairs) - (n - new) // BLOCK)
            pairs += [(b, block) for block in range((n - new) // BLOCK, (n - 1) // BLOCK + 1)]
        pairs = np.array(pairs)
        state["pair_page"] = torch.from_numpy(
            table[pairs[:, 0], pairs[:, 1] * BLOCK // page].astype(np.int64)).to(dev)
        state["pair_block"] = torch.from_numpy(pairs[:, 1] % (page // BLOCK)).to(dev)
        begin = (np.array(lengths) - np.array(news))[pairs[:, 0]]
        state["pair_kept"] = torch.from_numpy(np.maximum(0, begin - pairs[:, 1] * BLOCK)).to(dev)
        state["row_pair"] = torch.from_numpy(np.array(first)[seq] + position // BLOCK).to(dev)
    else:
        state["k_out"] = torch.empty((total, heads, dim), dtype=dtype, device=dev)
        state["v_out"] = torch.empty((total, heads, dim), dtype=dtype, device=dev)
    return state


# --------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return _own(state, op)
    if op == "attention":
        return _plain_attention(state)
    if op == "write":
        return _plain_write(state)
    if op == "read":
        return _plain_read(state)
    return _plain_rotary(state)


def _cache_outputs(state):
    """The cache as the numbers it stands for: E4M3 values and power-of-two scales."""
    return {"k_values": state["k_values"].view(torch.float8_e4m3fn),
            "v_values": state["v_values"].view(torch.float8_e4m3fn),
            "k_scales": state["k_scales"].view(torch.float8_e8m0fnu),
            "v_scales": state["v_scales"].view(torch.float8_e8m0fnu)}


def _own(state, op):
    import mxfp6_sm120_b200 as mxfp6

    if op == "rotary":
        return mxfp6.rotary_multi_axis(
            state["q"], state["k"], state["positions"],
            mxfp6.RotaryFrequencies(state["inv_freq"], state["axis"]),
            q_out=state["q_out"], k_out=state["k_out"])
    cache = mxfp6.PagedKVCache(state["k_values"], state["v_values"], state["k_scales"],
                               state["v_scales"])
    if op == "attention":
        return mxfp6.kv_cache_attention(
            state["q"], cache, state["table"], state["lengths"], state["starts"],
            max_query_len=state["widest"], causal=state["case"]["causal"], out=state["out"])
    if op == "write":
        mxfp6.kv_cache_write(cache, state["k"], state["v"], state["table"], state["lengths"],
                             state["starts"])
        return _cache_outputs(state)
    return mxfp6.kv_cache_read(cache, state["table"], state["lengths"], state["starts"],
                               out=(state["k_out"], state["v_out"]))


def _power(exponent):
    """2^exponent of whole numbers -126..127 in 32 bits, from the exponent field: no rounding."""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _decoded(values, scales, table, longest):
    """Pages of every sequence as 32-bit ``[batch, heads, longest, dim]``."""
    pages = table.clamp(min=0).long()
    codes = values[pages].view(torch.float8_e4m3fn).float()      # [B, P, H, page, D]
    b, p, h, page, d = codes.shape
    factor = _power(scales[pages].int() - 127)                   # [B, P, H, page / 32]
    codes = codes.view(b, p, h, page // BLOCK, BLOCK, d) * factor[..., None, None]
    return codes.permute(0, 2, 1, 3, 4, 5).reshape(b, h, p * page, d)[:, :, :longest]


def _plain_attention(state):
    case, q = state["case"], state["q"]
    batch, widest, longest = case["batch"], state["widest"], state["longest"]
    heads, dim = case["kv_heads"], case["dim"]
    group = case["q_heads"] // heads
    k = _decoded(state["k_values"], state["k_scales"], state["table"], longest)
    v = _decoded(state["v_values"], state["v_scales"], state["table"], longest)
    at = torch.arange(longest, device=q.device)
    held = at[None, :] < state["lengths"][:, None]               # [B, L]
    k = torch.where(held[:, None, :, None], k, 0.0)
    v = torch.where(held[:, None, :, None], v, 0.0)
    # rows of the batch padded to the widest sequence
    rows = torch.zeros((batch, widest, heads, group, dim), device=q.device)
    rows[state["seq"], state["index"]] = q.float().view(-1, heads, group, dim)
    place = torch.zeros((batch, widest), dtype=torch.long, device=q.device)
    place[state["seq"], state["index"]] = state["position"]
    rows = rows.permute(0, 2, 3, 1, 4).reshape(batch, heads, group * widest, dim)
    scores = rows @ k.transpose(2, 3) * (1.0 / math.sqrt(dim))
    scores = scores.view(batch, heads, group, widest, longest)
    allowed = held[:, None, :].expand(batch, widest, longest)
    if case["causal"]:
        allowed = allowed & (at[None, None, :] <= place[:, :, None])
    scores = torch.where(allowed[:, None, None], scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(batch, heads, group * widest, longest) @ v).view(
        batch, heads, group, widest, dim) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(batch, widest, heads * group, dim)
    return out[state["seq"], state["index"]].to(q.dtype)


def _plain_write(state):
    for source, values, scales in ((state["k"], state["k_values"], state["k_scales"]),
                                   (state["v"], state["v_values"], state["v_scales"])):
        page, block = state["pair_page"], state["pair_block"]
        p, h, size, d = values.shape
        blocks = values.view(p, h, size // BLOCK, BLOCK, d)
        old = blocks[page, :, block].view(torch.float8_e4m3fn).float()       # [N, H, 32, D]
        kept = state["pair_kept"][:, None]                                   # tokens already there
        slot = state["position"] % BLOCK
        fresh = torch.zeros_like(old)
        fresh[state["row_pair"], :, slot] = source.float()
        new = torch.zeros(old.shape[0], BLOCK, dtype=torch.bool, device=old.device)
        new[state["row_pair"], slot] = True
        # smallest power of two that takes the largest new magnitude to 448 or less
        top = fresh.abs().amax((2, 3))
        mantissa, exponent = torch.frexp(top)                                # top = m * 2^e, m < 1
        need = torch.clamp(exponent - 1 - 8 + 127 + (mantissa * 2 > 1.75).int(), min=FLOOR_CODE)
        need = torch.where(top > 0, need, FLOOR_CODE)
        before = scales[page, :, block].int()
        code = torch.where(kept > 0, torch.maximum(before, need), need)
        moved = old * _power(before - code)[..., None, None]
        fresh = fresh * _power(127 - code)[..., None, None]
        value = torch.where(new[:, None, :, None], fresh, moved).clamp(-MAX_CODE, MAX_CODE)
        row = torch.arange(BLOCK, device=old.device)
        touched = new | (row[None, :] < kept)
        coded = value.to(torch.float8_e4m3fn).view(torch.uint8)
        same = blocks[page, :, block]
        # tokens behind the last new one stay as they were
        blocks[page, :, block] = torch.where(touched[:, None, :, None], coded, same)
        scales[page, :, block] = code.to(torch.uint8)
    return _cache_outputs(state)


def _plain_read(state):
    out = []
    for values, scales in ((state["k_values"], state["k_scales"]),
                           (state["v_values"], state["v_scales"])):
        rows = _decoded(values, scales, state["table"], state["longest"])
        rows = rows.permute(0, 2, 1, 3)[state["seq"], state["position"]]
        out.append(rows.to(_DTYPES[state["case"]["dtype"]]))
    return tuple(out)


def _plain_rotary(state):
    half = state["inv_freq"].numel()
    # far positions: the angle needs more bits than 32 have
    angle = state["positions"][state["axis"].long()].t().double() * state["inv_freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for x in (state["q"], state["k"]):
        y = x.float()
        a, b = y[..., :half], y[..., half : 2 * half]
        out.append(torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half :]], -1).to(x.dtype))
    return tuple(out)


# --------------------------------------------------------------------------- work


def work(case):
    """Bytes and operations that one pass cannot do without."""
    if case["op"] == "rotary":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]
        rotated = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["rotary_dim"]
        return {"bytes": 4 * values + 8 * case["axes"] * case["tokens"], "flops": 3 * rotated}
    lengths, news = _lengths(case)
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "write":
        blocks = sum((n - 1) // BLOCK - (n - new) // BLOCK + 1 for n, new in zip(lengths, news))
        return {"bytes": 2 * (sum(news) * row * 3 + blocks * case["kv_heads"]), "flops": 0}
    scales = 2 * case["kv_heads"] * sum(-(-n // BLOCK) for n in lengths)
    if case["op"] == "read":
        return {"bytes": 2 * sum(news) * row * 3 + scales, "flops": 0}
    queries = 2 * 2 * sum(news) * case["q_heads"] * case["dim"]
    pairs = 0
    for n, new in zip(lengths, news):
        pairs += new * n - (new * (new - 1) // 2 if case["causal"] else 0)
    return {"bytes": 2 * sum(lengths) * row + scales + queries,
            "flops": 4 * pairs * case["q_heads"] * case["dim"]}


# --------------------------------------------------------------------------- the definition in 64 bits


def _power64(exponent):
    """2^exponent of whole numbers in 64 bits, from the exponent field."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(x):
    """Nearest E4M3 value, ties to even, saturating; ``x`` in 64 bits."""
    x = x.clamp(-MAX_CODE, MAX_CODE)
    exponent = torch.frexp(x)[1] - 1
    step = _power64(torch.clamp(exponent, min=-6) - 3)
    return torch.round(x / step) * step


def _e4m3_of_codes(codes):
    """Value of each byte, from its fields."""
    codes = codes.int()
    sign = 1.0 - 2.0 * (codes >> 7).double()
    field, fraction = (codes >> 3) & 15, (codes & 7).double()
    value = torch.where(field > 0, (1 + fraction / 8) * _power64(field - 7),
                        fraction / 8 * 2.0 ** -6)
    return sign * torch.where((codes & 127) == 127, math.nan, value)


def _sequence(values, scales, pages, length, heads):
    """One sequence's tokens in 64 bits, ``[heads, length, dim]``."""
    page = values.shape[2]
    out = _e4m3_of_codes(values[pages.long()][:, heads])
    factor = _power64(scales[pages.long()][:, heads].long() - 127)
    out = out * factor.repeat_interleave(BLOCK, dim=-1)[..., None]
    return out.transpose(0, 1).reshape(len(heads), len(pages) * page, -1)[:, :length]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        half = case["rotary_dim"] // 2
        out = []
        for x in (state["q"].double(), state["k"].double()):
            y = x.clone()
            for i in range(half):
                theta = state["positions"][state["axis"][i]].double() * state["inv_freq"][i]
                c, s = torch.cos(theta)[:, None], torch.sin(theta)[:, None]
                y[..., i] = x[..., i] * c - x[..., half + i] * s
                y[..., half + i] = x[..., half + i] * c + x[..., i] * s
            out.append(y)
        return tuple(out)
    lengths, news = _lengths(case)
    page = case["page"]
    table = state["table"]
    if case["op"] == "read":
        out = []
        for name in ("k", "v"):
            rows = [_sequence(state[name + "_values"], state[name + "_scales"],
                              table[b, : -(-n // page)], n, list(range(case["kv_heads"])))
                    for b, n in enumerate(lengths)]
            out.append(torch.cat([r.transpose(0, 1) for r in rows]))
        return tuple(out)
    if case["op"] == "write":
        out = {}
        for name in ("k", "v"):
            source = state[name].double()
            held = _e4m3_of_codes(state[name + "_values"])
            scale = _power64(state[name + "_scales"].long() - 127)
            row = 0
            for b, (n, new) in enumerate(zip(lengths, news)):
                position = n - new
                while position < n:
                    end = min(n, position // BLOCK * BLOCK + BLOCK)
                    where, kept = int(table[b, position // page]), position % BLOCK
                    block = position % page // BLOCK
                    tokens = source[row : row + end - position].transpose(0, 1)      # [H, t, D]
                    top = tokens.abs().amax((1, 2))
                    least = _power64(torch.ceil(torch.log2(torch.clamp(top / MAX_CODE, min=1e-35))))
                    # the logarithm of an exact power may come out one step off
                    least = torch.where(top / (least / 2) <= MAX_CODE, least / 2, least)
                    least = torch.where(top / least > MAX_CODE, least * 2, least)
                    least = torch.clamp(least, min=2.0 ** (FLOOR_CODE - 127))
                    was = scale[where, :, block].clone()
                    now = torch.maximum(least, was) if kept else least
                    lo = block * BLOCK
                    if kept:
                        before = held[where, :, lo : lo + kept]
                        held[where, :, lo : lo + kept] = _round_e4m3(before * (was / now)[:, None, None])
                    held[where, :, lo + kept : lo + kept + end - position] = _round_e4m3(
                        tokens / now[:, None, None])
                    scale[where, :, block] = now
                    row += end - position
                    position = end
            out[name + "_values"], out[name + "_scales"] = held, scale
        return out
    # attention, one sequence and key head at a time
    heads, dim = case["kv_heads"], case["dim"]
    group = case["q_heads"] // heads
    out = torch.zeros((state["tokens"], case["q_heads"], dim), dtype=torch.float64, device="cuda")
    row = 0
    for b, (n, new) in enumerate(zip(lengths, news)):
        pages = table[b, : -(-n // page)]
        for h in range(heads):
            k = _sequence(state["k_values"], state["k_scales"], pages, n, [h])[0]
            v = _sequence(state["v_values"], state["v_scales"], pages, n, [h])[0]
            for g in range(h * group, (h + 1) * group):
                scores = state["q"][row : row + new, g].double() @ k.t() / math.sqrt(dim)
                if case["causal"]:
                    last = torch.arange(n - new, n, device="cuda")
                    later = torch.arange(n, device="cuda")[None, :] > last[:, None]
                    scores.masked_fill_(later, -math.inf)
                out[row : row + new, g] = torch.softmax(scores, -1) @ v
        row += new
    return out

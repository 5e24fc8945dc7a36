"""Cases of the quantised key/value cache: writing tokens into it, reading them back, attending to it.

A cache holds keys and values as unsigned codes of `bits` bits in groups of `group` values along the
head dimension, value = scale * code + bias, in pages of `page` token rows per key/value head:
codes [pages, kv_heads, page, head_dim * bits / 32] (32 / bits codes to a 32-bit word, the first in the
lowest bits), scales and biases [pages, kv_heads, page, head_dim / group].  A sequence's page list is a
row of the block table; without one, page b holds sequence b.

update     k, v [batch, kv_heads, tokens, head_dim] -> codes, scales and biases at positions
           offset .. offset + count, and the values that the cache now stands for.  Per group
           scale = max((max - min) / (2^bits - 1), 1e-8), bias = min, code = (x - bias) / scale to the
           nearest whole number; the differences and quotients of this line are rounded to 32 bits
           each, which decides what lies at a border between two codes
fetch      the cache's values as dense [batch, kv_heads, length, head_dim] arrays, zero behind a sequence
attend     softmax(scale * q k^T) v over the cache, grouped query heads, optionally causal with the
           last query at the sequence's last token
"""

import math

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# --------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------


def _update(name, batch, kv_heads, tokens, head_dim, dtype, group, bits, page, history, ragged):
    return {"name": name, "op": "update", "batch": batch, "kv_heads": kv_heads, "tokens": tokens,
            "head_dim": head_dim, "dtype": dtype, "group": group, "bits": bits, "page": page,
            "history": history, "ragged": ragged}


def _fetch(name, batch, kv_heads, length, head_dim, dtype, group, bits, page, ragged):
    return {"name": name, "op": "fetch", "batch": batch, "kv_heads": kv_heads, "length": length,
            "head_dim": head_dim, "dtype": dtype, "group": group, "bits": bits, "page": page,
            "ragged": ragged}


def _attend(name, batch, heads, kv_heads, tokens, length, head_dim, dtype, group, page, ragged, causal):
    return {"name": name, "op": "attend", "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "tokens": tokens, "length": length, "head_dim": head_dim, "dtype": dtype, "group": group,
            "bits": 4, "page": page, "ragged": ragged, "causal": causal}


def listed():
    return [
        # one new token of one sequence: what every decode step pays per layer, all latency
        _update("update_one_token", 1, 8, 1, 128, "bfloat16", 64, 4, 16, 1000, False),
        # drafted tokens of a ragged batch into an 8-bit cache, small heads, small groups
        _update("update_drafts_8bit", 16, 8, 37, 64, "float16", 32, 8, 16, 611, True),
        # prompts of the decoder configuration (32 heads of 128, 8192 tokens), whole batch at once
        _update("update_prompts", 4, 32, 8192, 128, "bfloat16", 64, 4, 64, 0, False),
        # a short history read back in 32 bits, odd length
        _fetch("fetch_short_f32", 1, 8, 501, 128, "float32", 32, 8, 16, False),
        # a ragged batch of histories read back for a dense attention kernel
        _fetch("fetch_batch", 16, 8, 8192, 128, "bfloat16", 64, 4, 64, True),
        # decode of a single short sequence: latency
        _attend("attend_one_token", 1, 32, 8, 1, 1000, 128, "bfloat16", 64, 16, False, False),
        # decode of a serving batch with lengths up to the decoder's 8192
        _attend("attend_batch", 64, 32, 8, 1, 8192, 128, "bfloat16", 64, 16, True, False),
        # decode of one very long sequence, in fp16: one row block, all parallelism along the keys
        _attend("attend_long", 1, 64, 8, 1, 131077, 128, "float16", 128, 256, False, False),
        # checking five drafted tokens of each sequence, small heads and groups, odd lengths
        _attend("attend_drafts", 16, 16, 2, 5, 2047, 64, "float16", 32, 16, True, True),
        # decode in 32 bits with wide heads, one query head to a cache head
        _attend("attend_f32", 4, 8, 8, 1, 2048, 256, "float32", 64, 32, True, False),
        # a chunk of a long prompt against its history and itself
        _attend("attend_chunk", 1, 32, 8, 2048, 8192, 128, "bfloat16", 64, 16, False, True),
        # whole prompts, no grouping of heads, the cache of each sequence in one piece
        _attend("attend_prompts", 2, 32, 32, 4096, 4096, 128, "bfloat16", 64, 0, False, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["update", "fetch", "attend", "attend"])
    head_dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 64, 128) if head_dim % g == 0])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    page = rng.choice([0, 8, 16, 16, 24, 64, 256])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 8, 16, 32])
    bits = rng.choice([4, 4, 8])
    ragged = rng.random() < 0.5
    rows = 262144 * 128 // (kv_heads * head_dim)  # token rows: at most a quarter of the largest listed cases'
    if op == "update":
        tokens = _log(rng, 1, 8192)
        batch = _log(rng, 1, max(1, min(128, rows // tokens)))
        return {"op": op, "batch": batch, "kv_heads": kv_heads, "tokens": tokens, "head_dim": head_dim,
                "dtype": dtype, "group": group, "bits": bits, "page": page,
                "history": rng.randrange(0, 2000), "ragged": ragged}
    if op == "fetch":
        length = _log(rng, 1, 16384)
        batch = _log(rng, 1, max(1, min(64, rows // length)))
        return {"op": op, "batch": batch, "kv_heads": kv_heads, "length": length, "head_dim": head_dim,
                "dtype": dtype, "group": group, "bits": bits, "page": page, "ragged": ragged}
    per = rng.choice([1, 2, 4, 4, 5, 8, 16])  # query heads to a cache head
    while per * kv_heads > 64:
        per = max(1, per // 2)
    # one token, a few drafted ones, or a chunk
    tokens = rng.choice([1, 1, 1, _log(rng, 2, 16), _log(rng, 17, 1024)])
    if dtype == "float32":
        tokens = min(tokens, 64)
    pairs = (1 << 28) // (per * kv_heads)  # queries x keys: at most the largest listed case's products
    length = _log(rng, tokens, max(tokens, min(65536, rows, pairs // tokens)))
    batch = _log(rng, 1, max(1, min(64, rows // length, pairs // (tokens * length))))
    return {"op": op, "batch": batch, "heads": per * kv_heads, "kv_heads": kv_heads, "tokens": tokens,
            "length": length, "head_dim": head_dim, "dtype": dtype, "group": group, "bits": 4,
            "page": page, "ragged": ragged, "causal": tokens > 1 and rng.random() < 0.8}


# --------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------


def _spread(n, batch, ragged):
    """A length for each sequence: all `n`, or spread evenly over 1 .. n in a mixed order."""
    if not ragged:
        return [n] * batch
    return [max(1, n * ((7 * b + 3) % batch + 1) // batch) for b in range(batch)]


def _plan(case):
    """Host-side lengths of a case: (new or queried tokens, tokens in the cache with them)."""
    if case["op"] == "update":
        counts = _spread(case["tokens"], case["batch"], case["ragged"])
        return counts, [h + c for h, c in zip(_spread(case["history"], case["batch"], case["ragged"]), counts)]
    lengths = _spread(case["length"], case["batch"], case["ragged"])
    return [min(case.get("tokens", 1), n) for n in lengths], lengths


def _normal(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _codes_of(x, group, bits):
    """(codes packed into 32-bit words, scales, biases) of x along its last axis, in 32 bits."""
    top = (1 << bits) - 1
    dtype = x.dtype
    g = x.float().unflatten(-1, (-1, group))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    # a divisor on the device: by a Python number torch multiplies with its rounded reciprocal
    scale = ((hi - lo) / torch.full((), float(top), device=x.device)).clamp_min(1e-8).to(dtype)
    bias = lo.to(dtype)
    code = torch.round((g - bias.float()) / scale.float()).nan_to_num(0.0).clamp(0, top).to(torch.int32)
    code = code.flatten(-2).unflatten(-1, (-1, 32 // bits))
    shift = torch.arange(0, 32, bits, device=x.device, dtype=torch.int32)
    return (code << shift).sum(-1, dtype=torch.int32), scale.squeeze(-1), bias.squeeze(-1)


def _values_of(codes, scales, biases, group, bits):
    """scale * code + bias in 32 bits."""
    shift = torch.arange(0, 32, bits, device=codes.device, dtype=torch.int32)
    code = ((codes.unsqueeze(-1) >> shift) & ((1 << bits) - 1)).flatten(-2).unflatten(-1, (-1, group))
    return (scales.float().unsqueeze(-1) * code.float() + biases.float().unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, dim, heads = _DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    counts, lengths = _plan(case)
    batch, longest = len(lengths), max(lengths)
    page = case["page"] or longest
    columns = -(-longest // page)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["page"]:
        # every sequence's pages lie anywhere; entries behind its last page hold -1
        needed = [-(-n // page) for n in lengths]
        pages = sum(needed) + 1
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((batch, columns), -1, dtype=torch.int32, device="cuda")
        used = 0
        for b, n in enumerate(needed):
            table[b, :n] = order[used:used + n]
            used += n
    else:
        pages, table = batch, None
    state = {"case": dict(case), "table": table, "lengths": ints(lengths), "counts": ints(counts),
             "offsets": ints([n - c for n, c in zip(lengths, counts)]), "longest": longest}
    cache = []
    for which in range(2):
        # keys carry a few channels of larger magnitude, as projections of real models do
        loud = torch.ones(dim, device="cuda")
        if which == 0:
            loud[torch.randperm(dim, generator=gen, device="cuda")[: dim // 32]] = 4.0
        parts = [torch.empty((pages, heads, page, dim * case["bits"] // 32), dtype=torch.int32, device="cuda")]
        parts += [torch.empty((pages, heads, page, dim // case["group"]), dtype=dtype, device="cuda") for _ in range(2)]
        step = max(1, (1 << 26) // (heads * page * dim))  # pages at a time: bounds the 32-bit temporaries
        for at in range(0, pages, step):
            x = _normal((min(step, pages - at), heads, page, dim), gen, torch.float32) * loud
            for part, new in zip(parts, _codes_of(x.to(dtype), case["group"], case["bits"])):
                part[at:at + step] = new
        cache.append(tuple(parts))
    state["keys"], state["values"] = cache
    if case["op"] == "update":
        shape = (batch, heads, case["tokens"], dim)
        state["k"], state["v"] = _normal(shape, gen, dtype), _normal(shape, gen, dtype)
    elif case["op"] == "attend":
        state["q"] = _normal((batch, case["heads"], case["tokens"], dim), gen, dtype)
        state["scale"] = dim ** -0.5
    if own:
        # the handles that a program keeps beside its cache: the same tensors, wrapped
        from phew_b200 import mx

        state["cache"] = mx.fast.QuantizedKVCache(tuple(mx.array(t) for t in state["keys"]),
                                                  tuple(mx.array(t) for t in state["values"]),
                                                  group_size=case["group"], bits=case["bits"])
        state["mx"] = {n: None if state.get(n) is None else mx.array(state[n])
                       for n in ("table", "lengths", "counts", "offsets", "k", "v", "q")}
    return state


# --------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        return {"update": _own_update, "fetch": _own_fetch, "attend": _own_attend}[op](state)
    return {"update": _plain_update, "fetch": _plain_fetch, "attend": _plain_attend}[op](state)


def _own_update(state):
    from phew_b200 import mx

    a = state["mx"]
    k, v = mx.fast.quantized_cache_update(state["cache"], a["k"], a["v"], a["offsets"], block_table=a["table"],
                                          counts=a["counts"], fetch=True)
    return {"k": k._t, "v": v._t, "k_scales": state["keys"][1], "k_biases": state["keys"][2],
            "v_scales": state["values"][1], "v_biases": state["values"][2]}


def _own_fetch(state):
    from phew_b200 import mx

    a = state["mx"]
    k, v = mx.fast.quantized_cache_fetch(state["cache"], a["lengths"], block_table=a["table"],
                                         max_length=state["longest"])
    return {"k": k._t, "v": v._t}


def _own_attend(state):
    from phew_b200 import mx

    a = state["mx"]
    o = mx.fast.quantized_cache_attention(a["q"], state["cache"], a["lengths"], block_table=a["table"],
                                          counts=a["counts"], scale=state["scale"],
                                          mask="causal" if state["case"]["causal"] else None)
    return {"o": o._t}


def _rows(state, positions):
    """(page, row in the page) of token positions [batch, n]; positions behind a sequence give page 0."""
    page = state["keys"][0].shape[2]
    if state["table"] is None:
        index = torch.arange(positions.shape[0], device="cuda").unsqueeze(1).expand_as(positions)
        return index, positions.clamp_max(page - 1)
    column = (positions // page).clamp_max(state["table"].shape[1] - 1)
    return state["table"].long().gather(1, column).clamp_min(0), positions % page


def _plain_update(state):
    case = state["case"]
    token = torch.arange(case["tokens"], device="cuda")
    live = token < state["counts"].unsqueeze(1)
    pages, rows = _rows(state, state["offsets"].long().unsqueeze(1) + token)
    seq, tok = live.nonzero(as_tuple=True)
    at = pages[seq, tok], slice(None), rows[seq, tok]
    k = _plain_write(case, state["k"], state["keys"], live, seq, tok, at)
    v = _plain_write(case, state["v"], state["values"], live, seq, tok, at)
    return {"k": k, "v": v, "k_scales": state["keys"][1], "k_biases": state["keys"][2],
            "v_scales": state["values"][1], "v_biases": state["values"][2]}


def _plain_write(case, x, parts, live, seq, tok, at):
    """Writes x's live tokens into one side of the cache; the values that they now stand for."""
    codes, scales, biases = _codes_of(x, case["group"], case["bits"])
    parts[0][at] = codes.transpose(1, 2)[seq, tok]
    parts[1][at] = scales.transpose(1, 2)[seq, tok]
    parts[2][at] = biases.transpose(1, 2)[seq, tok]
    values = _values_of(codes, scales, biases, case["group"], case["bits"])
    return torch.where(live[:, None, :, None], values, 0.0).to(x.dtype)


def _dense(state, parts):
    """A cache side as dense 32-bit values [batch, kv_heads, longest, head_dim]."""
    positions = torch.arange(state["longest"], device="cuda").expand(len(state["lengths"]), -1)
    pages, rows = _rows(state, positions)
    picked = [p[pages, :, rows].transpose(1, 2) for p in parts]
    return _values_of(*picked, state["case"]["group"], state["case"]["bits"])


def _plain_fetch(state):
    live = torch.arange(state["longest"], device="cuda") < state["lengths"].unsqueeze(1)
    live = live[:, None, :, None]
    return {name: torch.where(live, _dense(state, parts), 0.0).to(parts[1].dtype)
            for name, parts in (("k", state["keys"]), ("v", state["values"]))}


def _plain_attend(state):
    case, q = state["case"], state["q"]
    batch, heads, tokens, dim = q.shape
    per = heads // case["kv_heads"]
    k, v = _dense(state, state["keys"]), _dense(state, state["values"])
    key = torch.arange(state["longest"], device="cuda")
    token = torch.arange(tokens, device="cuda")
    lengths, counts = state["lengths"].unsqueeze(1), state["counts"].unsqueeze(1)
    seen = (key < lengths)[:, None, :] & (token < counts)[:, :, None]
    if case["causal"]:
        seen = seen & (key <= (lengths - counts + token)[:, :, None])
    seen = seen[:, None, None]
    grouped = q.float().unflatten(1, (case["kv_heads"], per))
    s = (grouped.flatten(2, 3) @ k.transpose(-1, -2)).unflatten(2, (per, tokens))
    s = (s * state["scale"]).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (per, tokens)) / total.clamp_min(torch.finfo(torch.float32).tiny)
    return {"o": torch.where(seen.any(-1, keepdim=True), o, 0.0).flatten(1, 2).to(q.dtype)}


# --------------------------------------------------------------------------------------------------
# work and the exact result
# --------------------------------------------------------------------------------------------------


def work(case):
    counts, lengths = _plan(case)
    size = 4 if case["dtype"] == "float32" else 2
    dim, heads, batch = case["head_dim"], case["kv_heads"], case["batch"]
    packed = dim * case["bits"] // 8 + 2 * size * (dim // case["group"])  # a row of keys or values
    lists = 4 * batch + (4 * sum(-(-n // case["page"]) for n in lengths) if case["page"] else 0)
    if case["op"] == "update":
        new = sum(counts) * heads
        dense = batch * case["tokens"] * heads * dim * size  # what fetch=True writes, padded rows too
        return {"bytes": 2 * (new * (dim * size + packed) + dense) + lists, "flops": 2 * new * dim * 6}
    if case["op"] == "fetch":
        return {"bytes": 2 * (sum(lengths) * heads * packed + batch * max(lengths) * heads * dim * size) + lists,
                "flops": 2 * sum(lengths) * heads * dim * 2}
    pairs = sum(c * n - (c * (c - 1) // 2 if case["causal"] else 0) for c, n in zip(counts, lengths))
    queries = batch * case["heads"] * case["tokens"] * dim * size
    return {"bytes": 2 * sum(lengths) * heads * packed + 2 * queries + lists,
            "flops": 4 * pairs * case["heads"] * dim}


def _sequence64(state, parts, b, length):
    """Sequence b of a cache side, [kv_heads, length, head_dim] in 64 bits, page by page."""
    case = state["case"]
    codes, scales, biases = parts
    page, got = codes.shape[2], []
    for column in range(-(-length // page)):
        at = b if state["table"] is None else int(state["host_table"][b][column])
        got.append(tuple(p[at, :, : min(page, length - column * page)] for p in parts))
    codes, scales, biases = (torch.cat(x, dim=1) for x in zip(*got))
    per, top = 32 // case["bits"], 1 << case["bits"]
    words = codes.to(torch.int64) & 0xFFFFFFFF
    digits = []
    for _ in range(per):
        digits.append(words % top)
        words = words // top
    value = torch.stack(digits, dim=-1).reshape(*codes.shape[:2], -1).double()
    value *= scales.double().repeat_interleave(case["group"], dim=-1)
    return value + biases.double().repeat_interleave(case["group"], dim=-1)


def exact(case, seed):
    counts, lengths = _plan(case)
    state = prepare(case, seed)
    state["host_table"] = None if state["table"] is None else state["table"].cpu().tolist()
    if case["op"] == "update":
        return _exact_update(state, counts)
    longest = max(lengths)
    if case["op"] == "fetch":
        out = {}
        for name, parts in (("k", state["keys"]), ("v", state["values"])):
            rows = torch.zeros(len(lengths), case["kv_heads"], longest, case["head_dim"], dtype=torch.float64,
                               device="cuda")
            for b, n in enumerate(lengths):
                rows[b, :, :n] = _sequence64(state, parts, b, n)
            out[name] = rows
        return out
    q = state["q"].double()
    per = case["heads"] // case["kv_heads"]
    o = torch.zeros_like(q)
    for b, (c, n) in enumerate(zip(counts, lengths)):
        k, v = _sequence64(state, state["keys"], b, n), _sequence64(state, state["values"], b, n)
        for h in range(case["heads"]):
            s = torch.mm(q[b, h, :c], k[h // per].T) * state["scale"]
            if case["causal"]:
                later = torch.arange(n, device="cuda")[None, :] - torch.arange(c, device="cuda")[:, None] > n - c
                s[later] = -math.inf
            o[b, h, :c] = torch.mm(torch.softmax(s, dim=-1), v[h // per])
    return {"o": o}


def _to32(x):
    """x rounded to 32 bits, kept in 64 (a quotient of 32-bit numbers rounds there as in 32 bits)."""
    return x.float().double()


def _exact_update(state, counts):
    case, dtype = state["case"], state["k"].dtype
    page = state["keys"][0].shape[2]
    top = 2 ** case["bits"] - 1
    out = {}
    for name, x, parts in (("k", state["k"], state["keys"]), ("v", state["v"], state["values"])):
        groups = x.double().reshape(*x.shape[:-1], -1, case["group"])
        low = groups.min(dim=-1).values
        # the cache keeps the scale in its own type, and codes are taken against the kept scale
        step = _to32(_to32(groups.max(dim=-1).values - low) / top).clamp(min=_to32(1e-8 + torch.zeros_like(low)))
        step = step.to(dtype).double()
        code = torch.round(_to32(_to32(groups - low[..., None]) / step[..., None])).clamp(0, top)
        values = (code * step[..., None] + low[..., None]).reshape(x.shape)
        scales, biases = parts[1].double(), parts[2].double()
        for b, c in enumerate(counts):
            values[b, :, c:] = 0.0
            first = int(state["offsets"][b])
            done = 0
            while done < c:
                column, row = divmod(first + done, page)
                n = min(page - row, c - done)
                at = b if state["table"] is None else int(state["host_table"][b][column])
                scales[at, :, row:row + n] = step[b, :, done:done + n]
                biases[at, :, row:row + n] = low[b, :, done:done + n]
                done += n
        out[name], out[name + "_scales"], out[name + "_biases"] = values, scales, biases
    return out

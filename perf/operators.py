"""The key/value cache operators, measured: quantising rows as they are written
and reading them back, attention over the cache, and attention of a batch that
shares a prefix.

A case names one operator (``op``), the cache's format (f16, q8 or q4), its
head layout (``q_heads``, ``kv_heads``, ``head_dim``), its page size, the batch
and ``tokens``, the new tokens of each sequence.  Sequence lengths lie between
``shortest`` and ``longest``, spread evenly (the golden-ratio sequence), so
that they are known from the case alone.
"""
import math

import torch

own = False

QMAX = {"q8": 127.0, "q4": 7.0}
BLOCK = 32  # values under one scale of the q4 format; q8 has one scale for a head
GOLDEN = 0.6180339887498949


# --------------------------------------------------------------------- cases

def _case(name, op, fmt, batch, tokens, shortest, longest, q_heads=32, kv_heads=8, head_dim=128, page=64, prefix=0,
          source="f16", result="f16"):
    return dict(name=name, op=op, format=fmt, batch=batch, tokens=tokens, shortest=shortest, longest=longest,
                q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, page=page, prefix=prefix, source=source,
                result=result)


def listed():
    return [
        # one decode step of a batch: the new token's k and v enter the cache (f16 projections)
        _case("write_decode_q8", "write", "q8", 32, 1, 100, 4000),
        # a 1024-pixel image's tokens at once, from f32 projections, 4 bits a value
        _case("write_prompt_q4", "write", "q4", 1, 4352, 4352, 4352, source="f32"),
        # short odd prompts of the image model's head layout, kept for an f32 consumer
        _case("write_odd_q8", "write", "q8", 5, 37, 37, 300, 28, 7, 120, 16, source="f32", result="f32"),
        # whole contexts widened for a consumer of contiguous f16 k and v
        _case("read_batch_q8", "read", "q8", 8, 4352, 4000, 4352),
        # a few odd contexts of 120-value heads, widened to f32
        _case("read_odd_q4", "read", "q4", 3, 1001, 700, 1001, 28, 7, 120, 16, result="f32"),
        # the smallest decode step: one sequence, a short context
        _case("decode_one_q8", "attention", "q8", 1, 1, 1000, 1000),
        # a serving batch of ragged contexts in 4 bits
        _case("decode_batch_q4", "attention", "q4", 64, 1, 300, 8192),
        # an unquantised cache of 64-value heads
        _case("decode_f16_d64", "attention", "f16", 16, 1, 3000, 4352, 16, 8, 64),
        # six drafted tokens a sequence, checked at once; odd contexts, 120-value heads
        _case("draft_batch_q8", "attention", "q8", 16, 6, 501, 2600, 28, 7, 120, 16),
        # a chunk of a long prompt against what is already cached
        _case("chunk_q8", "attention", "q8", 1, 512, 8704, 8704),
        # a small batch behind a short instruction template
        _case("prefix_small_q4", "prefix", "q4", 8, 1, 1, 200, prefix=1024),
        # a large batch behind a long shared document
        _case("prefix_large_q8", "prefix", "q8", 128, 1, 16, 512, prefix=16384),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "prefix"])
    fmt = rng.choice(["q8", "q4", "f16", "q8", "q4"])
    kv_heads = rng.choice([1, 2, 4, 7, 8])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 8])
    head_dim = rng.choice([64, 72, 96, 120, 128, 128, 128])
    page = rng.choice([16, 32, 48, 64, 64, 128, 256])
    source, result = rng.choice(["f16", "f32"]), rng.choice(["f16", "f32"])
    prefix = 0
    if op in ("write", "read"):
        tokens = _log(rng, 1, 4352)
        batch = _log(rng, 1, max(1, min(64, 14000 // tokens)))
        longest = tokens + _log(rng, 1, 1000) - 1
        shortest = tokens if op == "write" else rng.randint(0, longest)
    else:
        result = "f16"
        tokens = rng.choice([1, 1, 1, 2, 5, 8, 16, _log(rng, 16, 512)])
        batch = _log(rng, 1, max(1, min(128, 512 // tokens)))
        held = {"f16": 80000, "q8": 150000, "q4": 280000}[fmt]  # rows of about one size in bytes
        room = max(64, min(16384, held // batch, 1000000 // (tokens * batch)))
        if op == "prefix":
            prefix = _log(rng, 1, room)
            room = max(tokens, min(room, 512, 60000 // batch))
        longest = _log(rng, min(tokens, room), max(tokens, room))
        longest = max(longest, tokens)
        shortest = rng.randint(tokens, longest)
    return {k: v for k, v in _case("", op, fmt, batch, tokens, shortest, longest, q_heads, kv_heads, head_dim, page,
                                   prefix, source, result).items() if k != "name"}


def _lengths(case):
    lo, hi, n = case["shortest"], case["longest"], case["batch"]
    if n == 1:
        return [hi]
    return [lo + int((hi - lo + 1) * ((i * GOLDEN) % 1.0)) for i in range(n)]


def _starts(case):
    """First position that a read takes: a write is read back where it went, a context from its first row."""
    return [length - case["tokens"] if case["op"] == "write" else 0 for length in _lengths(case)]


def _row_bytes(case):
    """Bytes of one token's k or v of one head in the cache, scales included."""
    d = case["head_dim"]
    return {"f16": 2 * d, "q8": d + 2, "q4": d / 2 + 2 * math.ceil(d / BLOCK)}[case["format"]]


def work(case):
    b, s, d, hq, hkv = (case[k] for k in ("batch", "tokens", "head_dim", "q_heads", "kv_heads"))
    row, lengths = _row_bytes(case), _lengths(case)
    width = {"f16": 2, "f32": 4}
    if case["op"] in ("write", "read"):
        rows = 2 * hkv * sum(max(0, min(s, n - a)) for n, a in zip(lengths, _starts(case)))
        out = 2 * hkv * b * s * d * width[case["result"]]
        if case["op"] == "write":
            return {"bytes": rows * (d * width[case["source"]] + 2 * row) + out, "flops": 4 * rows * d}
        return {"bytes": rows * row + out, "flops": rows * d}
    seen = sum(sum(max(0, n - s + i + 1) for i in range(s)) for n in lengths) + b * s * case["prefix"]
    kv = 2 * hkv * (sum(lengths) + case["prefix"]) * row
    return {"bytes": kv + 2 * 2 * b * s * hq * d, "flops": 4 * hq * d * seen}


# --------------------------------------------------------------------- inputs

def _rows(shape, head_axis, generator):
    """k or v rows as projections give them: noise of unit size over per-channel offsets of each head."""
    offset_shape = [1] * len(shape)
    offset_shape[head_axis], offset_shape[-1] = shape[head_axis], shape[-1]
    offsets = torch.randn(offset_shape, generator=generator, device="cuda")
    return torch.randn(shape, generator=generator, device="cuda").add_(offsets, alpha=0.6)


def _quantise(x, fmt):
    """Whole numbers (in f32) and scales of rows x [..., D] in f32."""
    d = x.shape[-1]
    block = d if fmt == "q8" else BLOCK
    pad = -d % block
    blocks = torch.nn.functional.pad(x, (0, pad)).reshape(*x.shape[:-1], (d + pad) // block, block)
    top = blocks.abs().amax(-1, keepdim=True)
    scale = (top / torch.full((), QMAX[fmt], device=x.device)).to(torch.bfloat16).float()
    q = torch.where(scale > 0, (blocks / scale).round().clamp(-QMAX[fmt], QMAX[fmt]), torch.zeros_like(blocks))
    return q.reshape(*x.shape[:-1], d + pad)[..., :d], scale[..., 0]


def _widen(q, scale, fmt):
    """Rows in f32 from stored values and scales."""
    if fmt == "f16":
        return q.float()
    d = q.shape[-1]
    per = scale.repeat_interleave(d if fmt == "q8" else BLOCK, -1)[..., :d]
    return q.float() * per


def _store(x, fmt):
    """What the cache holds of rows x: stored values (f16, or int8 whole numbers) and scales."""
    if fmt == "f16":
        return x.half(), None
    q, scale = _quantise(x.float(), fmt)
    return q.to(torch.int8), scale


def _dtype(name):
    return {"f16": torch.float16, "f32": torch.float32}[name]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    b, s, hkv, d, page, fmt = (case[k] for k in ("batch", "tokens", "kv_heads", "head_dim", "page", "format"))
    lengths = _lengths(case)
    width = max(1, -(-max(lengths) // page))
    shared = -(-case["prefix"] // page)
    pages = b * width + shared
    order = torch.randperm(pages, generator=host).to(device="cuda", dtype=torch.int32)  # pages in no order
    state = dict(case=case, table=order[:b * width].reshape(b, width).contiguous(),
                 prefix_table=order[b * width:].contiguous(),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                 starts=torch.tensor(_starts(case), dtype=torch.int32, device="cuda"),
                 prefix_length=torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda"))
    if case["op"] == "write":
        state["key"] = _rows((b, s, hkv, d), 2, g).to(_dtype(case["source"]))
        state["value"] = _rows((b, s, hkv, d), 2, g).to(_dtype(case["source"]))
        if not own:
            kind = torch.float16 if fmt == "f16" else torch.int8
            blocks = 1 if fmt == "q8" else -(-d // BLOCK)
            for name in ("k", "v"):
                state[name] = torch.zeros((pages, page, hkv, d), dtype=kind, device="cuda")
                state[name + "_scale"] = torch.zeros((pages, page, hkv, blocks), device="cuda")
    else:
        # every page is full of rows; those behind a sequence's length are another's leavings
        rows = {name: _rows((pages, page, hkv, d), 2, g).half() for name in ("k", "v")}
        if not own:
            for name, x in rows.items():
                state[name], state[name + "_scale"] = _store(x, fmt)
    if case["op"] in ("attention", "prefix"):
        state["query"] = torch.randn((b, s, case["q_heads"], d), generator=g, device="cuda").half()
    if own:
        from burn_image_b200 import KVCache
        state["cache"] = cache = KVCache(pages, page, hkv, d, fmt)
        if case["op"] != "write":
            every = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(pages, 1)
            cache.append(rows["k"], rows["v"], every, torch.full((pages,), page, dtype=torch.int32, device="cuda"))
        state["longest"] = max(lengths)
    return state


# --------------------------------------------------------------------- one pass

def _slots(state, positions):
    """Pool rows (page, place) of positions [B, n], with those out of range taken at row 0."""
    page, table = state["case"]["page"], state["table"].long()
    inside = positions.clamp(0, table.shape[1] * page - 1)
    return torch.gather(table, 1, inside // page), inside % page


def _take(state, name, pages, places):
    scale = state[name + "_scale"]
    return _widen(state[name][pages, places], None if scale is None else scale[pages, places], state["case"]["format"])


def _plain_write(state):
    case = state["case"]
    positions = state["starts"].long()[:, None] + torch.arange(case["tokens"], device="cuda")
    pages, places = _slots(state, positions)
    for name, x in (("k", state["key"]), ("v", state["value"])):
        q, scale = _store(x, case["format"])
        state[name][pages, places] = q
        if scale is not None:
            state[name + "_scale"][pages, places] = scale


def _plain_read(state):
    case = state["case"]
    positions = state["starts"].long()[:, None] + torch.arange(case["tokens"], device="cuda")
    pages, places = _slots(state, positions)
    held = ((positions >= 0) & (positions < state["lengths"][:, None]))[:, :, None, None]
    zero = torch.zeros((), device="cuda")
    return tuple(torch.where(held, _take(state, name, pages, places), zero).transpose(1, 2).contiguous()
                 .to(_dtype(case["result"])) for name in ("k", "v"))


def _softmax_parts(scores, visible, values):
    """Row maximum, sum and unnormalised product of one set of keys."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-1e30)
    weights = (scores - top).exp()
    return top, weights.sum(-1, keepdim=True), weights @ values


def _plain_attention(state):
    case = state["case"]
    b, s, hq, hkv, d = (case[k] for k in ("batch", "tokens", "q_heads", "kv_heads", "head_dim"))
    group = hq // hkv
    q = state["query"].float().reshape(b, s, hkv, group, d).permute(0, 2, 1, 3, 4) / math.sqrt(d)  # [B, Hkv, S, G, D]
    longest = state["table"].shape[1] * case["page"]
    positions = torch.arange(longest, device="cuda").expand(b, longest)
    pages, places = _slots(state, positions)
    k, v = (_take(state, name, pages, places).transpose(1, 2) for name in ("k", "v"))  # [B, Hkv, L, D]
    last = state["lengths"].long()[:, None] - s + torch.arange(s, device="cuda") + 1  # keys that query i sees
    visible = (positions[:, None] < last[:, :, None])[:, None, :, None].expand(b, 1, s, group, longest)
    scores = q.reshape(b, hkv, s * group, d) @ k.transpose(-1, -2)
    # a row behind the length holds anything; it must not reach the sums
    v = v.masked_fill((positions >= state["lengths"][:, None])[:, None, :, None], 0.0)
    top, total, out = _softmax_parts(scores, visible.reshape(b, 1, s * group, longest), v)
    if case["op"] == "prefix":
        n = case["prefix"]
        places = torch.arange(n, device="cuda")
        pages = state["prefix_table"].long()[places // case["page"]]
        places = places % case["page"]
        pk, pv = (_take(state, name, pages, places).transpose(0, 1) for name in ("k", "v"))  # [Hkv, P, D]
        rows = q.permute(1, 0, 2, 3, 4).reshape(hkv, b * s * group, d)
        every = torch.ones((), dtype=torch.bool, device="cuda").expand(hkv, b * s * group, n)
        parts = _softmax_parts(rows @ pk.transpose(-1, -2), every, pv)
        ptop, ptotal, pout = (x.reshape(hkv, b, s * group, -1).transpose(0, 1) for x in parts)
        both = torch.maximum(top, ptop)
        a, c = (top - both).exp(), (ptop - both).exp()
        total, out = total * a + ptotal * c, out * a + pout * c
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.reshape(b, hkv, s, group, d).permute(0, 2, 1, 3, 4).reshape(b, s, hq, d).half()


def run(state):
    case = state["case"]
    if own:
        cache = state["cache"]
        if case["op"] in ("write", "read"):
            if case["op"] == "write":
                cache.append(state["key"], state["value"], state["table"], state["lengths"])
            return cache.read(state["table"], state["lengths"], case["tokens"], starts=state["starts"],
                              dtype=_dtype(case["result"]))
        if case["op"] == "prefix":
            return cache.prefix_attention(state["query"], state["prefix_table"], state["prefix_length"], state["table"],
                                          state["lengths"], max_length=state["longest"])
        return cache.attention(state["query"], state["table"], state["lengths"], max_length=state["longest"])
    if case["op"] == "write":
        _plain_write(state)
    return _plain_attention(state) if case["op"] in ("attention", "prefix") else _plain_read(state)


# --------------------------------------------------------------------- 64 bits

def _held64(rows, fmt):
    """The values that the cache stands for, of rows [..., D], in 64 bits: the scale is the bf16 nearest to the f32
    quotient of the largest magnitude and the largest whole number, the whole number the one nearest to the f32
    quotient of value and scale."""
    if fmt == "f16":
        return rows.half().double()
    x = rows.double()
    d, top = x.shape[-1], QMAX[fmt]
    parts = []
    for part in x.split(d if fmt == "q8" else BLOCK, dim=-1):
        scale = (part.abs().amax(-1, keepdim=True) / top).float().bfloat16().double()
        whole = torch.nan_to_num(part / scale).float().double().round().clamp(-top, top)
        parts.append(whole * scale)
    return torch.cat(parts, -1)


def exact(case, seed):
    b, s, hkv, d, page, fmt = (case[k] for k in ("batch", "tokens", "kv_heads", "head_dim", "page", "format"))
    lengths = _lengths(case)
    if case["op"] in ("attention", "prefix") and case["q_heads"] * s * b * (max(lengths) + case["prefix"]) * d > 2e12:
        return None
    g = torch.Generator(device="cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    width = max(1, -(-max(lengths) // page))
    shared = -(-case["prefix"] // page)
    order = torch.randperm(b * width + shared, generator=host)
    if case["op"] == "write":
        made = [_rows((b, s, hkv, d), 2, g).to(_dtype(case["source"])) for _ in range(2)]
        return tuple(_held64(x, fmt).transpose(1, 2).contiguous() for x in made)
    key, value = (_rows((b * width + shared, page, hkv, d), 2, g).half() for _ in range(2))
    query = None if case["op"] == "read" else torch.randn((b, s, case["q_heads"], d), generator=g, device="cuda").half()

    def context(x, pages, n):  # the first n rows of a page list, [Hkv, n, D]
        return _held64(x[pages.cuda()].reshape(-1, hkv, d)[:n], fmt).transpose(0, 1)

    if case["op"] == "read":
        outs = []
        for x in (key, value):
            out = torch.zeros((b, hkv, s, d), dtype=torch.float64, device="cuda")
            for i, n in enumerate(lengths):
                n = min(n, s)
                out[i, :, :n] = context(x, order[i * width:(i + 1) * width], n)
            outs.append(out)
        return tuple(outs)
    group = case["q_heads"] // hkv
    out = torch.zeros((b, s, case["q_heads"], d), dtype=torch.float64, device="cuda")
    before = [context(x, order[b * width:], case["prefix"]) for x in (key, value)]
    for i, n in enumerate(lengths):
        mine = order[i * width:(i + 1) * width]
        k, v = (torch.cat([p, context(x, mine, n)], 1) for p, x in zip(before, (key, value)))
        first = case["prefix"] + n - s + 1
        for h in range(hkv):
            rows = query[i, :, h * group:(h + 1) * group].double()  # [S, G, D]
            scores = torch.einsum("sgd,nd->sgn", rows, k[h]) / math.sqrt(d)
            hidden = torch.arange(k.shape[1], device="cuda")[None, :] >= first + torch.arange(s, device="cuda")[:, None]
            weights = torch.softmax(scores.masked_fill(hidden[:, None], -math.inf), -1)
            out[i, :, h * group:(h + 1) * group] = torch.einsum("sgn,nd->sgd", weights, v[h])
    return torch.where(out.isnan(), torch.zeros_like(out), out)

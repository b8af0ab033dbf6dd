"""The work that the operators for a cache in 4 bits and for scoring tokens are measured on.

Four operators, as a program that serves or scores text calls them: a step's keys and values go into a paged
cache of 4-bit codes and are read back as the values held (``write``), single tokens attend over that cache
(``decode``), prompt portions attend over it (``prompt``), and logits rows give the log probability of a given token
with the row's entropy, the token's rank and the most likely alternatives (``logprobs``).

The cache: 32 consecutive head dimensions of one key (or value) form a group with one step ``d``.  With ``e`` the
element of largest magnitude (the positive one where both signs have it), ``d`` is ``-e / 8`` rounded to five
significant bits, and an element is held as ``code = clamp(rint(x / d), -8, 7) + 8``, which stands for
``(code - 8) d``.  A page of one head holds the codes of its keys, ``16 G`` bytes each for ``G`` groups, then their
steps, ``G`` bfloat16 each.  In a key's row the 32-bit word ``c G + g`` holds dimensions ``32 g + 8 c ..+ 7``, lowest bits
first; in a value's row the byte ``n G + g`` holds dimensions ``32 g + 2 n`` and the next one."""

import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
GROUP = 32


def _kernels():
    from pagedserve_amd.ops import kernels

    return kernels


# ------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the write of a decode step: 8 requests, GPT-2 small's heads
        {"name": "write step of 8", "op": "write", "items": 8, "tokens": 8, "kv_heads": 12, "dim": 64, "page": 16,
         "type": "bfloat16", "lengths_seed": 1},
        # a prompt step's write: 2 x 1,024 tokens, GPT-2 XL's 25 heads
        {"name": "write 2 x 1024, 25 heads", "op": "write", "items": 2, "tokens": 2048, "kv_heads": 25, "dim": 64,
         "page": 16, "type": "bfloat16", "lengths_seed": 2},
        # a ragged portion in 32-bit, heads whose last group is half full
        {"name": "write 301 float, heads of 48", "op": "write", "items": 3, "tokens": 301, "kv_heads": 5, "dim": 48,
         "page": 8, "type": "float32", "lengths_seed": 3},
        # one user, GPT-2 small near the end of its context
        {"name": "decode 1 x 900", "op": "decode", "items": 1, "shortest": 900, "longest": 900, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "type": "bfloat16", "window": 0, "lengths_seed": 4},
        # the XL workload: 64 requests between their prompt's end and 1,024
        {"name": "decode 64 x 768..1024, 25 heads", "op": "decode", "items": 64, "shortest": 768, "longest": 1024,
         "heads": 25, "kv_heads": 25, "dim": 64, "page": 16, "type": "bfloat16", "window": 0, "lengths_seed": 5},
        # long contexts: 32 requests over 8,192 keys each
        {"name": "decode 32 x 8192", "op": "decode", "items": 32, "shortest": 8192, "longest": 8192, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "type": "bfloat16", "window": 0, "lengths_seed": 6},
        # grouped heads of 128, ragged contexts of thousands of keys
        {"name": "decode 24 x 500..6000, 16 / 2 heads", "op": "decode", "items": 24, "shortest": 500, "longest": 6000,
         "heads": 16, "kv_heads": 2, "dim": 128, "page": 32, "type": "bfloat16", "window": 0, "lengths_seed": 7},
        # the true 32-bit path
        {"name": "decode 8 x 540 float", "op": "decode", "items": 8, "shortest": 100, "longest": 540, "heads": 12,
         "kv_heads": 12, "dim": 64, "page": 16, "type": "float32", "window": 0, "lengths_seed": 8},
        # whole prompts, 2 x 1,024 tokens of GPT-2 small
        {"name": "prompt 2 x 1024", "op": "prompt", "items": 2, "shortest": 1024, "longest": 1024, "start": 0,
         "heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "type": "bfloat16", "window": 0, "lengths_seed": 9},
        # later portions of long prompts, grouped heads of 128
        {"name": "prompt portions behind 5000, 16 / 4 heads", "op": "prompt", "items": 3, "shortest": 150,
         "longest": 512, "start": 5000, "heads": 16, "kv_heads": 4, "dim": 128, "page": 16, "type": "bfloat16",
         "window": 0, "lengths_seed": 10},
        # a decode step's rows, each with its token and five alternatives
        {"name": "logprobs 8 x 50257, top 5", "op": "logprobs", "rows": 8, "vocab": 50257, "top": 5,
         "type": "float32", "masked": 0},
        # scoring a prompt portion, twenty alternatives a token
        {"name": "logprobs 512 x 50257, top 20", "op": "logprobs", "rows": 512, "vocab": 50257, "top": 20,
         "type": "float32", "masked": 0},
    ]


def _log_between(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """Another case of those ranges: heads of 16 to 256, groups of 1 to 16 heads, pages of 8 to 64 keys, 1 to 64
    requests, contexts of one key to 8,192, prompts of one token to 1,024, both types, windows; up to 600 rows of 300 to
    160,000 logits."""
    op = rng.choice(("write", "decode", "decode", "prompt", "logprobs"))
    seed = rng.randrange(1 << 30)
    if op == "logprobs":
        vocab = _log_between(rng, 300, 160000)
        rows = _log_between(rng, 1, min(600, 25_000_000 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "top": rng.choice((0, 1, 3, 8, 20)),
                "type": rng.choice(("float32", "float32", "bfloat16")), "masked": rng.choice((0, 0, 1)), "lengths_seed": seed}
    kv_heads, group = rng.choice(((12, 1), (25, 1), (16, 1), (2, 8), (4, 4), (5, 3), (1, 16), (8, 2)))
    case = {"op": op, "kv_heads": kv_heads, "dim": rng.choice((16, 48, 64, 64, 96, 128, 128, 256)),
            "page": rng.choice((8, 16, 16, 32, 64)), "type": rng.choice(("bfloat16", "bfloat16", "float32")), "lengths_seed": seed}
    if op == "write":
        items = rng.randint(1, 16)
        case.update(items=items, tokens=_log_between(rng, items, 2048))
        return case
    case.update(heads=kv_heads * group, window=rng.choice((0, 0, 0, 200)))
    if op == "decode":
        items = _log_between(rng, 1, 64)
        longest = _log_between(rng, 1, min(8192, 50_000_000 // (items * case["heads"] * case["dim"])))
        case.update(items=items, shortest=max(1, longest // rng.choice((1, 2, 8))), longest=longest)
        return case
    case["type"] = "bfloat16"
    items = rng.randint(1, 4)
    longest = _log_between(rng, 2, 1024)
    case.update(items=items, shortest=max(1, longest // 3), longest=longest, start=rng.choice((0, 0, 37, 700, 2000)))
    return case


# ------------------------------------------------------------------------------------- the cache's form
def _groups(case):
    return -(-case["dim"] // GROUP)


def _lengths(case):
    """Tokens that every request brings (``write``, ``prompt``) or has (``decode``), from the case alone."""
    rng = random.Random(case["lengths_seed"])
    items = case["items"]
    if case["op"] == "write":
        cuts = sorted(rng.sample(range(1, case["tokens"]), items - 1)) if items > 1 else []
        return [b - a for a, b in zip([0] + cuts, cuts + [case["tokens"]])]
    return [rng.randint(case["shortest"], case["longest"]) for _ in range(items)]


def _starts(case):
    if case["op"] == "write":
        rng = random.Random(case["lengths_seed"] + 1)
        return [rng.randint(0, 900) for _ in range(case["items"])]
    start = case.get("start", 0)
    return [start + 13 * i for i in range(case["items"])]


def _coded(x):
    """(codes as integers, steps) of groups ``x[..., 32]``."""
    x = x.to(F32)
    high, low = x.amax(-1), -x.amin(-1)
    step = torch.where(high >= low, high, -low) * -0.125
    bits = step.view(torch.int32)
    bits = (bits + 0x3ffff + ((bits >> 19) & 1)) & ~0x7ffff
    step = bits.view(F32)
    step = torch.where(step.abs() < 2.0 ** -126, torch.zeros_like(step), step)
    # (the quotient in 64 bits: a value next to the border of two codes falls on its own side)
    ratio = x.double() / torch.where(step == 0, torch.ones_like(step), step).double().unsqueeze(-1)
    codes = torch.where(step.unsqueeze(-1) == 0, torch.zeros_like(ratio), ratio.round().clamp(-8, 7))
    return codes.to(torch.int32) + 8, step


def _in_groups(x, case):
    """Rows ``[n, kv_heads * dim]`` as ``[n, kv_heads, G, 32]``, zeros behind the last dimension."""
    n, groups = x.shape[0], _groups(case)
    out = x.new_zeros((n, case["kv_heads"], groups * GROUP))
    out[..., :case["dim"]] = x.view(n, case["kv_heads"], case["dim"])
    return out.view(n, case["kv_heads"], groups, GROUP)


def _key_bytes(codes):
    """Codes ``[..., G, 32]`` as a key's row of bytes."""
    pairs = codes[..., 0::2] | (codes[..., 1::2] << 4)                       # [..., G, 16]
    words = pairs.unflatten(-1, (4, 4))                                      # [..., G, c, byte]
    return words.transpose(-3, -2).flatten(-3).to(torch.uint8)


def _value_bytes(codes):
    pairs = codes[..., 0::2] | (codes[..., 1::2] << 4)                       # [..., G, n]
    return pairs.transpose(-2, -1).flatten(-2).to(torch.uint8)


def _codes_of(rows, groups, keys):
    """Bytes ``[..., 16 G]`` of rows as codes ``[..., G, 32]``."""
    if keys:
        pairs = rows.unflatten(-1, (4, groups, 4)).transpose(-3, -2).flatten(-2)
    else:
        pairs = rows.unflatten(-1, (16, groups)).transpose(-2, -1)
    pairs = pairs.to(torch.int32)
    return torch.stack((pairs & 15, pairs >> 4), -1).flatten(-2)


def _held(pool, pages, case, keys):
    """The values in pages of a pool, ``[..., kv_heads, page, dim]`` in 32 bits (exact)."""
    groups, page = _groups(case), case["page"]
    raw = pool[pages].flatten(-2)                                            # [..., kv_heads, page bytes]
    codes = _codes_of(raw[..., :page * 16 * groups].unflatten(-1, (page, 16 * groups)), groups, keys)
    steps = raw[..., page * 16 * groups:].contiguous().view(torch.bfloat16).unflatten(-1, (page, groups))
    values = (codes - 8).to(F32) * steps.to(F32).unsqueeze(-1)
    return values.flatten(-2)[..., :case["dim"]]


def _new_pool(values, case, keys):
    """A pool whose pages hold ``values`` [pages, kv_heads, page, G, 32]."""
    codes, steps = _coded(values)
    rows = _key_bytes(codes) if keys else _value_bytes(codes)
    raw = torch.cat((rows.flatten(-2), steps.to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)), -1)
    return raw.view(values.shape[0], case["kv_heads"], case["page"], 18 * _groups(case)).contiguous()


def _dtype(case):
    return torch.bfloat16 if case["type"] == "bfloat16" else F32


# ------------------------------------------------------------------------------------------- prepare
def _pages(case, lengths, g):
    """Block tables for requests of those lengths over shuffled pages, and the number of pages."""
    needed = [-(-length // case["page"]) for length in lengths]
    width = max(needed) + 1
    order = torch.randperm(sum(needed) + 3, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for item, count in enumerate(needed):
        tables[item, :count] = order[at:at + count]
        at += count
    return tables, sum(needed) + 3


def _cache(case, pages, g):
    """Both pools full of keys and values: normal ones, some of the keys' dimensions several times as large."""
    shape = (pages, case["kv_heads"], case["page"], _groups(case) * GROUP)
    size = torch.ones(shape[-1], device="cuda")
    size[3::29] = 4.0
    pools = []
    for keys in (True, False):
        pool = torch.empty(shape[:3] + (18 * _groups(case),), dtype=torch.uint8, device="cuda")
        for at in range(0, pages, 2048):
            values = torch.randn((min(2048, pages - at),) + shape[1:], generator=g, device="cuda")
            if keys:
                values *= size
            values[..., case["dim"]:] = 0
            pool[at:at + values.shape[0]] = _new_pool(values.unflatten(-1, (_groups(case), GROUP)), case, keys)
        pools.append(pool)
    return pools


def _tiles(counts, starts, size):
    """The queries of portions in tiles, those that see the most keys first."""
    listed = [(start + q0, item, q0) for item, (count, start) in enumerate(zip(counts, starts))
              for q0 in range(0, count, size)]
    listed.sort(key=lambda tile: -tile[0])
    return (torch.tensor([t[1] for t in listed], dtype=torch.int32, device="cuda"),
            torch.tensor([t[2] for t in listed], dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _dtype(case)
    state = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.5
        likely = torch.randint(0, vocab, (rows, 12), generator=g, device="cuda")
        logits.scatter_add_(1, likely, torch.rand((rows, 12), generator=g, device="cuda") * 9.0)
        if case["masked"]:
            # tokens that the caller has forbidden
            logits[:, torch.randperm(vocab, generator=g, device="cuda")[:vocab // 50]] = -math.inf
        tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        tokens[::2] = likely[::2, 0]
        # (a token that was given was not forbidden)
        logits.scatter_(1, tokens[:, None], logits.gather(1, tokens[:, None]).clamp(min=-20.0))
        # (rows start at multiples of 8 values, as the engine's do)
        wide = torch.zeros((rows, -(-vocab // 8) * 8), dtype=kind, device="cuda")
        wide[:, :vocab] = logits.to(kind)
        state.update(logits=wide[:, :vocab], tokens=tokens.to(torch.int32))
        if own:
            state.update(
                out=torch.empty(rows, device="cuda"), entropy=torch.empty(rows, device="cuda"),
                ranks=torch.empty(rows, dtype=torch.int32, device="cuda"),
                top_ids=torch.empty((rows, top), dtype=torch.int32, device="cuda"),
                top_logprobs=torch.empty((rows, top), device="cuda"),
                partial=torch.empty(_kernels().logprob_scratch(rows, vocab, top), device="cuda"))
        return state
    counts, starts = _lengths(case), _starts(case)
    if case["op"] == "decode":
        lengths, counts, starts = counts, [1] * len(counts), [length - 1 for length in counts]
    else:
        lengths = [a + b for a, b in zip(counts, starts)]
    tables, pages = _pages(case, lengths, g)
    k_pool, v_pool = _cache(case, pages, g)
    tokens = sum(counts)
    tok_item = torch.tensor([i for i, n in enumerate(counts) for _ in range(n)], dtype=torch.int32, device="cuda")
    tok_pos = torch.tensor([s + j for n, s in zip(counts, starts) for j in range(n)], dtype=torch.int32, device="cuda")
    state.update(tables=tables, k_pool=k_pool, v_pool=v_pool, tok_item=tok_item, tok_pos=tok_pos, counts=counts,
                 starts=starts, lengths=lengths)
    if case["op"] == "write":
        # keys and values are columns of the packed projection's rows
        qkv = torch.randn((tokens, 3 * case["kv_heads"] * case["dim"]), generator=g, device="cuda")
        qkv[:, case["kv_heads"] * case["dim"]::29] *= 4.0
        qkv = qkv.to(kind)
        _, state["k"], state["v"] = qkv.split(case["kv_heads"] * case["dim"], dim=1)
        state["k_held"] = torch.empty((tokens, case["kv_heads"] * case["dim"]), dtype=kind, device="cuda")
        state["v_held"] = torch.empty_like(state["k_held"])
        return state
    heads, dim = case["heads"], case["dim"]
    state["q"] = torch.randn((tokens, heads * dim), generator=g, device="cuda").to(kind)
    state["scale"] = dim ** -0.5
    state["out"] = torch.zeros((tokens, heads * dim), dtype=kind, device="cuda")
    if case["op"] == "decode":
        if own:
            splits = _kernels().int4_decode_splits(kind, case["items"], heads, case["kv_heads"], dim,
                                                   min(max(lengths), case["window"] or max(lengths)))
            state["splits"] = splits
            state["partial"] = torch.empty(case["items"] * heads * splits * (dim + 2), device="cuda")
        return state
    state["cu_tokens"] = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    state["kv_lens"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    state["tiles"] = {size: _tiles(counts, starts, size) for size in (32, 64, 128)}
    return state


# ----------------------------------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    return {"write": _write, "decode": _decode, "prompt": _prompt, "logprobs": _logprobs}[case["op"]](case, state)


def _write(case, state):
    k, v, k_pool, v_pool = state["k"], state["v"], state["k_pool"], state["v_pool"]
    tok_item, tok_pos, tables = state["tok_item"], state["tok_pos"], state["tables"]
    if own:
        kernels = _kernels()
        kernels.kv_write_int4(k, v, k_pool, v_pool, tok_item, tok_pos, tables)
        kernels.kv_read_int4(k_pool, v_pool, state["k_held"], state["v_held"], tok_item, tok_pos, tables)
        return state["k_held"], state["v_held"]
    groups, page = _groups(case), case["page"]
    pages = tables[tok_item.long(), (tok_pos // page).long()].long()
    at = (tok_pos % page).long()
    held = []
    for x, pool, keys in ((k, k_pool, True), (v, v_pool, False)):
        codes, steps = _coded(_in_groups(x, case))
        flat = pool.flatten(2)                                               # [pages, kv_heads, page bytes]
        rows = flat[:, :, :page * 16 * groups].unflatten(-1, (page, 16 * groups))
        rows[pages, :, at] = _key_bytes(codes) if keys else _value_bytes(codes)
        places = flat[:, :, page * 16 * groups:].unflatten(-1, (page, 2 * groups))
        places[pages, :, at] = steps.to(torch.bfloat16).contiguous().view(torch.uint8)
        codes = _codes_of(rows[pages, :, at], groups, keys)
        steps = places[pages, :, at].contiguous().view(torch.bfloat16)
        values = (codes - 8).to(F32) * steps.to(F32).unsqueeze(-1)
        held.append(values.flatten(-2)[..., :case["dim"]].flatten(1).to(k.dtype))
    return tuple(held)


def _decode(case, state):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    q, tables, tok_pos = state["q"], state["tables"], state["tok_pos"]
    if own:
        _kernels().attention_decode_int4(
            q, state["k_pool"], state["v_pool"], state["out"], None, tok_pos, tables, heads, state["scale"],
            state["splits"], partial=state["partial"], window=case["window"])
        return state["out"]
    items, width = tables.shape
    pages = tables.clamp(min=0).long()
    k = _held(state["k_pool"], pages, case, True).transpose(1, 2).reshape(items, kv_heads, -1, dim)
    v = _held(state["v_pool"], pages, case, False).transpose(1, 2).reshape(items, kv_heads, -1, dim)
    queries = q.to(F32).view(items, kv_heads, heads // kv_heads, dim)
    scores = torch.matmul(queries, k.transpose(2, 3).contiguous()) * state["scale"]
    keys = torch.arange(k.shape[2], device=q.device)
    seen = keys[None] <= tok_pos[:, None]
    if case["window"]:
        seen &= keys[None] > tok_pos[:, None] - case["window"]
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.matmul(weights, v) / weights.sum(-1, keepdim=True)
    return out.reshape(items, heads * dim).to(q.dtype)


def _prompt(case, state):
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    q = state["q"]
    if own:
        kernels = _kernels()
        size = kernels.prefill_int4_tile(heads, dim, {n: t[0].numel() for n, t in state["tiles"].items()},
                                         max(state["lengths"]))
        kernels.attention_prefill_int4(
            q, state["k_pool"], state["v_pool"], state["out"], *state["tiles"][size], state["cu_tokens"],
            state["kv_lens"], state["tables"], heads, state["scale"], window=case["window"],
            max_kv_len=max(state["lengths"]), query_tile=size)
        return state["out"]
    out = torch.empty_like(q)
    first = 0
    for item, (count, start) in enumerate(zip(state["counts"], state["starts"])):
        pages = state["tables"][item, :-(-(start + count) // case["page"])].long()
        k = _held(state["k_pool"], pages, case, True).transpose(0, 1).reshape(kv_heads, -1, dim)
        v = _held(state["v_pool"], pages, case, False).transpose(0, 1).reshape(kv_heads, -1, dim)
        k, v = k[:, :start + count], v[:, :start + count]
        queries = q[first:first + count].to(F32).view(count, kv_heads, heads // kv_heads, dim)
        queries = queries.permute(1, 2, 0, 3).reshape(kv_heads, -1, dim)
        scores = torch.matmul(queries, k.transpose(1, 2).contiguous()) * state["scale"]
        scores = scores.view(kv_heads, heads // kv_heads, count, start + count)
        keys = torch.arange(start + count, device=q.device)
        places = torch.arange(start, start + count, device=q.device)
        seen = keys[None] <= places[:, None]
        if case["window"]:
            seen &= keys[None] > places[:, None] - case["window"]
        scores = scores.masked_fill(~seen, -math.inf)
        weights = torch.exp(scores - scores.amax(-1, keepdim=True))
        sums = weights.sum(-1, keepdim=True)
        mixed = torch.matmul(weights.view(kv_heads, -1, start + count), v).view(kv_heads, heads // kv_heads, count, dim)
        out[first:first + count] = (mixed / sums).permute(2, 0, 1, 3).reshape(count, heads * dim).to(q.dtype)
        first += count
    return out


def _logprobs(case, state):
    logits, tokens, top = state["logits"], state["tokens"], case["top"]
    if own:
        _kernels().token_logprobs(
            logits, tokens, state["out"], entropy=state["entropy"], ranks=state["ranks"],
            top_ids=state["top_ids"] if top else None, top_logprobs=state["top_logprobs"] if top else None,
            partial=state["partial"])
        found = (state["out"], state["entropy"], state["ranks"])
        return found + (state["top_ids"], state["top_logprobs"]) if top else found
    x = logits.to(F32)
    vocab = x.shape[1]
    highest = x.amax(-1, keepdim=True)
    shifted = x - highest
    weights = torch.exp(shifted)
    total = weights.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = log_total - torch.where(weights > 0, weights * shifted, torch.zeros_like(x)).sum(-1, keepdim=True) / total
    given = x.gather(1, tokens.long()[:, None])
    ids = torch.arange(vocab, device=x.device)
    ahead = (x > given) | ((x == given) & (ids < tokens[:, None]))
    found = ((given - highest - log_total)[:, 0], entropy[:, 0], ahead.sum(-1, dtype=torch.int32))
    if not top:
        return found
    # one whole number per logit, ordered as the logits are and unlike any other: the lower id first among equals
    bits = (x + 0.0).contiguous().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 20) + (vocab - 1 - ids)
    best = torch.topk(order, top, dim=-1).values
    top_ids = vocab - 1 - (best & ((1 << 20) - 1))
    return found + (top_ids.to(torch.int32), shifted.gather(1, top_ids) - log_total)


# --------------------------------------------------------------------------------------------- exact
def _number(code_bytes, low):
    return ((code_bytes.double() % 16 if low else torch.floor(code_bytes.double() / 16)) - 8.0)


def _exact_values(pool, pages, case, keys):
    """[kv_heads, len(pages) * page, dim] in 64 bits, dimension by dimension."""
    groups, page, dim = _groups(case), case["page"], case["dim"]
    raw = pool[pages].reshape(len(pages), case["kv_heads"], -1)
    rows = raw[..., :page * 16 * groups].reshape(len(pages), case["kv_heads"], page, 16 * groups)
    steps = raw[..., page * 16 * groups:].contiguous().view(torch.bfloat16).double()
    steps = steps.reshape(len(pages), case["kv_heads"], page, groups)
    out = torch.empty(rows.shape[:3] + (dim,), dtype=F64, device=pool.device)
    for d in range(dim):
        g, within = divmod(d, GROUP)
        at = 4 * ((within // 8) * groups + g) + (within % 8) // 2 if keys else (within // 2) * groups + g
        out[..., d] = _number(rows[..., at], d % 2 == 0) * steps[..., g]
    return out.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, dim)


def _exact_rounded(x):
    """What the cache holds of groups [..., n] in 64 bits."""
    largest = x.abs().amax(-1, keepdim=True)
    sign = torch.where((x == largest).any(-1, keepdim=True), 1.0, -1.0).double()
    mantissa, exponent = torch.frexp(largest / 8)
    step = -sign * torch.ldexp(torch.round(mantissa * 32) / 32, exponent)
    step = torch.where(step.abs() < 2.0 ** -126, torch.zeros_like(step), step)
    held = torch.round(x / torch.where(step == 0, torch.ones_like(step), step)).clamp(-8, 7) * step
    return held


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "write":
        found = []
        for x in (state["k"], state["v"]):
            heads = x.double().reshape(x.shape[0], case["kv_heads"], case["dim"])
            held = torch.cat([_exact_rounded(part) for part in heads.split(GROUP, dim=-1)], dim=-1)
            found.append(held.reshape(x.shape[0], -1))
        return tuple(found)
    if case["op"] == "logprobs":
        x = state["logits"].double()
        tokens = state["tokens"].long()
        log_p = x - torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(log_p)
        entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(-1)
        order = torch.sort(log_p, dim=-1, descending=True, stable=True).indices
        ranks = (order == tokens[:, None]).int().argmax(-1).to(torch.int32)
        found = (log_p.gather(1, tokens[:, None])[:, 0], entropy, ranks)
        if not case["top"]:
            return found
        best = order[:, :case["top"]]
        return found + (best.to(torch.int32), log_p.gather(1, best))
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    q = state["q"].double()
    out = torch.empty_like(q)
    first = 0
    for item, (count, start) in enumerate(zip(state["counts"], state["starts"])):
        length = start + count
        pages = state["tables"][item, :-(-length // case["page"])].long()
        keys = _exact_values(state["k_pool"], pages, case, True)
        values = _exact_values(state["v_pool"], pages, case, False)
        behind = torch.arange(start, length, device="cuda")[:, None] - torch.arange(length, device="cuda")[None]
        hidden = (behind < 0) | (behind >= (case["window"] or length + 1))
        for head in range(heads):
            kv = head // (heads // kv_heads)
            rows = q[first:first + count, head * dim:(head + 1) * dim]
            scores = rows @ keys[kv, :length].t().contiguous() * state["scale"]
            p = torch.softmax(scores.masked_fill(hidden, -math.inf), -1)
            out[first:first + count, head * dim:(head + 1) * dim] = p @ values[kv, :length]
        first += count
    return out


# ---------------------------------------------------------------------------------------------- work
def work(case):
    size = 2 if case["type"] == "bfloat16" else 4
    if case["op"] == "logprobs":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * size + case["rows"] * (16 + 8 * case["top"]), "flops": 8 * cells}
    held = 2 * case["kv_heads"] * 18 * _groups(case)          # bytes of one cached key and value
    if case["op"] == "write":
        values = 2 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": 2 * values * size + 2 * case["tokens"] * held, "flops": 6 * values}
    width = case["heads"] * case["dim"]
    counts, starts = _lengths(case), _starts(case)
    if case["op"] == "decode":
        counts, starts = [1] * len(counts), [length - 1 for length in counts]
    limit = case["window"] or (1 << 30)
    pairs = sum(min(start + j + 1, limit) for count, start in zip(counts, starts) for j in range(count))
    keys = sum(min(start + count, limit + count - 1) for count, start in zip(counts, starts))
    return {"bytes": keys * held + 2 * sum(counts) * width * size, "flops": 4 * pairs * width}

"""The cache in 4 bits from its definition, in 64 bits: what a group of 32 dimensions is held as, how a page's bytes
lie, attention over the values held with a bound of its float evaluation, and log probabilities."""

import math

import numpy as np
import torch

GROUP = 32


def step_of(group):
    """The step of a group of numbers (float64 array)."""
    if not np.isfinite(group).all():
        return float("nan")
    high, low = group.max(initial=0.0), group.min(initial=0.0)
    largest = high if high >= -low else low
    mantissa, exponent = math.frexp(-largest / 8.0)
    step = math.ldexp(np.rint(mantissa * 32.0) / 32.0, exponent)
    if abs(step) > 2.0 ** 125 * 31 / 32:                # the largest step whose eightfold is a float
        step = math.copysign(2.0 ** 125 * 31 / 32, step)
    return 0.0 if abs(step) < 2.0 ** -126 else step


def held(rows, kv_heads):
    """(codes [n, kv_heads, G, 32], steps [n, kv_heads, G], values [n, kv_heads * dim]) of rows [n, kv_heads * dim]."""
    rows = rows.double().cpu().numpy().reshape(rows.shape[0], kv_heads, -1)
    n, _, dim = rows.shape
    groups = -(-dim // GROUP)
    codes = np.full((n, kv_heads, groups, GROUP), 8, dtype=np.int64)
    steps = np.zeros((n, kv_heads, groups))
    values = np.zeros_like(rows)
    for t in range(n):
        for h in range(kv_heads):
            for g in range(groups):
                part = rows[t, h, g * GROUP:(g + 1) * GROUP]
                step = step_of(part)
                steps[t, h, g] = step
                if step != step:
                    values[t, h, g * GROUP:(g + 1) * GROUP] = np.nan
                    continue
                if step != 0.0:
                    codes[t, h, g, :part.size] = np.clip(np.rint(part / step), -8, 7).astype(np.int64) + 8
                values[t, h, g * GROUP:(g + 1) * GROUP] = (codes[t, h, g, :part.size] - 8) * step
    return codes, steps, torch.from_numpy(values.reshape(n, kv_heads * dim))


def row_bytes(codes, keys):
    """The bytes of one key's (or value's) row: codes [G, 32]."""
    groups = codes.shape[0]
    row = np.zeros(16 * groups, dtype=np.uint8)
    for g in range(groups):
        for d in range(GROUP):
            at = 4 * (d // 8 * groups + g) + d % 8 // 2 if keys else d // 2 * groups + g
            row[at] |= int(codes[g, d]) << 4 * (d % 2)
    return row


def store(pool, codes, steps, tables, items, positions, keys):
    """Write tokens into a pool of bytes [pages, kv_heads, page, 18 G] (a CPU tensor)."""
    pages, kv_heads, page_size, _ = pool.shape
    groups = steps.shape[2]
    flat = pool.view(pages, kv_heads, -1).numpy()
    for t, (item, position) in enumerate(zip(items, positions)):
        page, within = int(tables[item][position // page_size]), position % page_size
        for h in range(kv_heads):
            flat[page, h, within * 16 * groups:(within + 1) * 16 * groups] = row_bytes(codes[t, h], keys)
            bits = (torch.tensor(steps[t, h]).to(torch.bfloat16).view(torch.uint8)).numpy()
            at = page_size * 16 * groups + within * 2 * groups
            flat[page, h, at:at + 2 * groups] = bits


def visible(position, key, window):
    if key > position:
        return False
    if window > 0:
        return key > position - window
    if window < 0:
        return key >= position - position % -window
    return True


def _largest(x):
    """Every element of [.., dim] replaced by the largest magnitude of its group of 32."""
    return torch.cat([part.abs().amax(-1, keepdim=True).expand_as(part) for part in x.split(GROUP, dim=-1)], -1)


def attention(q, k, v, positions, heads, scale, window=0, sink=None, softcap=0.0):
    """(out, size, shift) in 64 bits for queries [n, heads * dim] at ``positions`` over the keys 0 .. of one request
    ([length, kv_heads * dim]).  ``size``: the weighted mean of the values' magnitudes and, for bfloat16 queries, 2^-7 of the weighted mean
    of their groups' largest ones: the kernels sum codes with an offset there, 16 + code less 24, at most 40 steps in any partial sum,
    where a group's largest value has 7 or more.  64 additions of a tile, rounded to 2^-24 of that, are
    64 * 40 / 7 * 2^-24 = 2^-15.5 of the largest value's share, and ``allowed`` takes 2^-8 of ``size``.  ``shift``: how far float evaluation may
    move a score (a sum of dim products, its scaling and the change to units of log 2), as an exponent."""
    n, length = q.shape[0], k.shape[0]
    offset = q.dtype == torch.bfloat16
    dim = q.shape[1] // heads
    kv_heads = k.shape[1] // dim
    q = q.double().cpu().view(n, heads, dim)
    k = k.double().cpu().view(length, kv_heads, dim)
    v = v.double().cpu().view(length, kv_heads, dim)
    mask = torch.tensor([[visible(p, j, window) for j in range(length)] for p in positions])
    out, size, shift = (torch.zeros(n, heads, dim, dtype=torch.float64) for _ in range(3))
    for h in range(heads):
        kh = k[:, h // (heads // kv_heads)]
        vh = v[:, h // (heads // kv_heads)]
        s = q[:, h] @ kh.T * scale
        absolute = q[:, h].abs() @ kh.nan_to_num(0.0).abs().T * abs(scale)
        if offset:      # (the same for the scores: partial sums of 40 steps to a query's element, a seventh of its group's largest key)
            absolute = absolute + q[:, h].abs() @ _largest(kh.nan_to_num(0.0)).T * abs(scale) * 40 / 7
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        s = s.masked_fill(~mask, -math.inf)
        moved = (2.0 ** -24 * ((dim + 8) * absolute + 8 * s.abs())).masked_fill(~mask, 0.0).amax(-1)
        if sink is not None:
            s = torch.cat((s, torch.full((n, 1), float(sink[h]), dtype=torch.float64)), -1)
        p = torch.softmax(s, -1)[:, :length]
        p = torch.where(mask, p, torch.zeros(()).double())
        seen = torch.where(mask.T[None], vh.T[:, :, None], torch.zeros(()).double())          # [dim, length, n]
        out[:, h] = torch.einsum("nl,dln->nd", p, seen)
        size[:, h] = torch.einsum("nl,dln->nd", p, seen.abs())
        if offset:
            large = torch.where(mask.T[None], _largest(vh).T[:, :, None], torch.zeros(()).double())
            size[:, h] += 2.0 ** -7 * torch.einsum("nl,dln->nd", p, large)
        shift[:, h] = moved[:, None]
    if sink is None:
        out[~mask.any(-1)] = 0.0
        size[~mask.any(-1)] = 0.0
    return (t.reshape(n, heads * dim) for t in (out, size, shift))


def allowed(out, size, shift, kind, weights):
    """How far a result may be off.  Scores moved by ``shift`` move every weight by as much of itself, the sum's too; weights
    rounded to bfloat16 (``weights``) move by half a step, 2^-8; the hardware's exponential is good to 2^-21 here; sums in float
    over thousands of keys add less than 2^-14 (the sums of integer codes, which carry an offset, among them); the result is rounded once."""
    rounding = 2.0 ** -8 if kind == torch.bfloat16 else 2.0 ** -24
    relative = 2 * shift + (2.0 ** -8 if weights else 0.0) + (2.0 ** -13 if kind == torch.bfloat16 else 2.0 ** -18)
    return size * relative + rounding * out.abs() + 1e-30


def logprobs(logits, tokens, top):
    """(log probability, entropy, rank, top ids, top log probabilities) in 64 bits."""
    x = logits.double().cpu()
    # (shifted first: next to 3.4e38 even 64 bits are 4e22 apart, and the logarithm of a sum would be lost)
    shifted = x - x.amax(-1, keepdim=True)
    log_p = shifted - torch.logsumexp(shifted, -1, keepdim=True)
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, torch.zeros(()).double()).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices
    tokens = tokens.long().cpu()
    rank = (order == tokens[:, None]).int().argmax(-1)
    ids = order[:, :top]
    return log_p.gather(1, tokens[:, None])[:, 0], entropy, rank, ids, log_p.gather(1, ids)

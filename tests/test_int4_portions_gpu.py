"""Prompt portions over a cache in 4 bits where a table or a page ends: against plain formulas in 64 bits."""

import math
from unittest import mock

import pytest
import torch

import plain_int4 as plain
from test_int4_gpu import _cache, _ints, _requests

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _portions(kind, dim, group=1):
    """(what it is, a call ``(q, pools, out, counts, lengths, tables, heads, window=0, sink=None)``) for every form of tile that
    takes the head size and as many heads to a key/value head, in one range and in several."""
    from pagedserve_amd.ops import kernels

    def call(size, name, **options):
        def run(q, pools, out, counts, lengths, tables, heads, window=0, sink=None):
            tiles = [(item, q0) for item, count in enumerate(counts) for q0 in range(0, count, size)]
            cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
            getattr(kernels, name)(q, *pools, out, _ints([t[0] for t in tiles]), _ints([t[1] for t in tiles]), _ints(cu),
                                   _ints(lengths), tables, heads, (q.shape[1] // heads) ** -0.5, window=window, sink=sink,
                                   query_tile=size, **options)
        return run

    if kind == F32:
        return [((size, paired), call(size, "attention_tiled_f32_int4", paired=paired))
                for size, paired in ((32, False), (64, False), (64, True))]
    sizes = (64, 128) if dim <= 128 else (64,)
    forms = [((size, ranges, most), call(size, "attention_prefill_int4", ranges=ranges, max_kv_len=most))
             for size in sizes for ranges, most in ((1, 0), (1, 100), (3, 0))]
    if group % 2 == 0 and 64 < dim <= 128:
        forms += [((64, ranges, "pairs"), call(64, "attention_prefill_int4", ranges=ranges, block_heads=2)) for ranges in (1, 3)]
    return forms


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("dim,page,width,window", [
    (64, 16, 7, 20), (64, 16, 7, 8), (64, 8, 13, -40), (128, 16, 5, 8), (128, 24, 3, -24), (256, 16, 7, 30), (48, 40, 2, 5),
    (64, 16, 7, 300), (16, 8, 3, -1000)])
def test_windows_that_begin_behind_the_table(kind, dim, page, width, window):
    """Portions whose last queries lie behind the block table, some by more than the window: those see nothing, and no
    entry of the table is asked for that is none."""
    if kind == F32 and dim > 128:
        pytest.skip("float portions of such heads go token by token")
    room = width * page
    starts = (max(0, room - 60), room - 3, room + 50)
    counts = (200, 70, 33)
    tables, pages, _, _ = _requests((1, 1, 1), (room - 1,) * 3, page, 15)
    tables = tables[:, :width].contiguous()
    pools, kept = _cache(tables, pages, (room,) * 3, 2, dim, page, 16)
    tokens = sum(counts)
    q = torch.randn((tokens, 2 * dim), generator=torch.Generator().manual_seed(17)).to(kind)
    positions = [start + j for start, count in zip(starts, counts) for j in range(count)]
    parts = [list(plain.attention(part, *kept[item], list(range(starts[item], starts[item] + counts[item])), 2, dim ** -0.5,
                                  window)) for item, part in enumerate(q.split(list(counts)))]
    expected = [torch.cat([part[which] for part in parts]) for which in range(3)]
    limit = plain.allowed(*expected, kind, kind == BF16)
    sees = torch.tensor([any(plain.visible(p, key, window) for key in range(room)) for p in positions])
    assert bool(sees.any()) and (window in (300, -1000) or not bool(sees.all()))
    for form, run in _portions(kind, dim):
        print(form, flush=True)
        out = torch.full((tokens + 1, 2 * dim), -9.0, dtype=kind).cuda()
        run(q.cuda(), pools, out[:tokens], counts, [a + b for a, b in zip(starts, counts)], tables.cuda(), 2, window)
        off = (out[:tokens].double().cpu() - expected[0]).abs() <= limit
        assert bool(off[sees].all()), form
        assert bool((out[tokens] == -9.0).all())


def _check(out, expected, kind, what):
    """NaN where the formula has one, and nowhere else; the rest within bounds."""
    out, limit = out.double().cpu(), plain.allowed(*expected, kind, kind == BF16)
    bad = expected[0].isnan()
    assert torch.equal(out.isnan(), bad), (what, (out.isnan() != bad).nonzero()[:4].tolist())
    assert bool(((out - expected[0]).abs()[~bad] <= limit[~bad]).all()), what


MISSING = [
    # group, dim, page, counts, starts, window, sink, logical pages of every request that the table does not have
    (1, 64, 16, (70,), (100,), 0, False, ((0, 4, 5, 9),)), (2, 128, 8, (66, 20), (30, 150), 0, False, ((1, 2, 11), (18, 19, 20, 21))),
    (1, 64, 24, (130, 3), (0, 50), 40, False, ((1, 4), (2,))), (2, 48, 16, (40, 33), (60, 0), 0, True, ((5,), (0, 1, 2))),
    (1, 256, 32, (70,), (200,), -64, False, ((3, 7),)), (2, 128, 64, (129,), (300,), 0, False, ((1, 5),)),
    (1, 16, 8, (65,), (8,), 0, False, (tuple(range(8)),))]


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("group,dim,page,counts,starts,window,sink,missing", MISSING)
def test_pages_that_the_table_does_not_have(kind, group, dim, page, counts, starts, window, sink, missing):
    """Keys whose entry lies outside the pool are seen by nobody, as single tokens have it: not those of another page."""
    from pagedserve_amd.ops import kernels

    if kind == F32 and dim > 128:
        pytest.skip("float portions of such heads go token by token")
    heads = 2 * group
    lengths = [a + b for a, b in zip(counts, starts)]
    tables, pages, items, positions = _requests(counts, starts, page, 81)
    pools, kept = _cache(tables, pages, lengths, 2, dim, page, 82)
    for item, gone in enumerate(missing):
        for turn, logical in enumerate(gone):
            tables[item, logical] = (-1, pages, 1 << 30)[turn % 3]
    q = torch.randn((sum(counts), heads * dim), generator=torch.Generator().manual_seed(83)).to(kind)
    sinks = torch.randn(heads, generator=torch.Generator().manual_seed(84)).cuda() if sink else None
    parts = []
    for item, part in enumerate(q.split(list(counts))):
        seen = plain.visible
        with mock.patch.object(plain, "visible", lambda at, key, window: seen(at, key, window)
                               and key // page not in missing[item]):
            parts.append(list(plain.attention(part, *kept[item], list(range(starts[item], lengths[item])), heads, dim ** -0.5,
                                              window, sinks)))
    expected = [torch.cat([part[which] for part in parts]) for which in range(3)]
    for form, run in _portions(kind, dim, group):
        print(form, flush=True)
        out = torch.full((len(items) + 1, heads * dim), -9.0, dtype=kind).cuda()
        run(q.cuda(), pools, out[:-1], counts, lengths, tables.cuda(), heads, window, sinks)
        blind = torch.cat([part[0] for part in parts]).eq(0).all(1)
        _check(out[:-1][~blind], [e[~blind] for e in expected], kind, form)
        assert bool((out[-1] == -9.0).all())
    out = torch.zeros((len(items), heads * dim), dtype=kind).cuda()
    kernels.attention_decode_int4(q.cuda(), *pools, out, _ints(items), _ints(positions), tables.cuda(), heads, dim ** -0.5, 1,
                                  None, window, sink=sinks)
    _check(out, expected, kind, "single tokens")

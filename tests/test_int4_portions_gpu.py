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


NO_NUMBER = [
    # group, dim, page, count, start, window, (position, head, group of dimensions; None: a key's) of what is no number
    (1, 64, 16, 70, 100, 0, ((3, 0, 1), (150, 1, 0))), (2, 128, 8, 66, 30, 0, ((95, 0, 3), (40, 1, 2), (41, 1, 0))),
    (1, 64, 24, 130, 0, 40, ((60, 0, 0), (61, 0, 1))), (2, 48, 16, 40, 60, 0, ((70, 1, 1), (99, 0, 0))),
    (1, 256, 32, 70, 200, -64, ((210, 0, 7), (255, 1, 4), (256, 1, 0))), (2, 128, 64, 129, 300, 0, ((310, 0, 1), (0, 1, 3))),
    (1, 16, 8, 65, 8, 0, ((20, 0, 0), (72, 1, 0))), (1, 96, 16, 50, 70, 0, ((90, 0, 2), (100, 0, None), (33, 1, 1))),
    (1, 32, 8, 70, 0, 0, ((0, 0, 0), (35, 1, None)))]


def _no_number(kind, group, dim, page, count, start, window, bad):
    from pagedserve_amd.ops import kernels

    heads, length = 2 * group, start + count
    tables, pages, items, positions = _requests((count,), (start,), page, 91)
    pools, ((k, v),) = _cache(tables, pages, (length,), 2, dim, page, 92)
    rows = [k.float(), v.float()]
    for position, head, which in bad:
        rows[which is not None][position, head * dim + 32 * (which or 0) + 5] = math.nan
    index = (_ints([0] * length), _ints(list(range(length))), tables.cuda())
    kernels.kv_write_int4(rows[0].cuda(), rows[1].cuda(), *pools, *index)
    kept = [plain.held(part, 2)[2] for part in rows]
    q = torch.randn((count, heads * dim), generator=torch.Generator().manual_seed(93)).to(kind)
    expected = list(plain.attention(q, *kept, positions, heads, dim ** -0.5, window))
    share = float(expected[0].isnan().double().mean())
    assert 0 < share < 0.9
    for form, run in _portions(kind, dim, group):
        print(form, flush=True)
        out = torch.full((count, heads * dim), -9.0, dtype=kind).cuda()
        run(q.cuda(), pools, out, (count,), (length,), tables.cuda(), heads, window)
        _check(out, expected, kind, form)
    out = torch.zeros((count, heads * dim), dtype=kind).cuda()
    kernels.attention_decode_int4(q.cuda(), *pools, out, _ints(items), _ints(positions), tables.cuda(), heads, dim ** -0.5, 1,
                                  None, window)
    _check(out, expected, kind, "single tokens")


@pytest.mark.parametrize("group,dim,page,count,start,window,bad", NO_NUMBER)
def test_what_is_no_number_stays_where_it_is(group, dim, page, count, start, window, bad):
    """A value's group that is no number makes these dimensions of its head so, for the queries that see it; a key, the head's."""
    _no_number(BF16, group, dim, page, count, start, window, bad)


def test_infinities_in_the_place_of_a_missing_page():
    """What nobody wrote may be anything, steps that are infinite among them, and page 0 may be such a page."""
    dim, page, count, start = 64, 16, 70, 40
    tables, pages, _, positions = _requests((count,), (start,), page, 85)
    tables[(tables >= 0) & (tables < pages)] += 1                           # (page 0 is nobody's)
    pools, ((k, v),) = _cache(tables, pages + 1, (start + count,), 2, dim, page, 86)
    for pool in pools:
        pool[0].view(2, -1)[:, page * 32:] = torch.tensor([0x80, 0x7f], dtype=torch.uint8).repeat(page * 2).cuda()
    tables[0, 3] = -1
    q = torch.randn((count, 2 * dim), generator=torch.Generator().manual_seed(87)).to(BF16)
    seen = plain.visible
    with mock.patch.object(plain, "visible", lambda at, key, window: seen(at, key, window) and key // page != 3):
        expected = list(plain.attention(q, k, v, positions, 2, dim ** -0.5))
    for form, run in _portions(BF16, dim):
        out = torch.full((count, 2 * dim), -9.0, dtype=BF16).cuda()
        run(q.cuda(), pools, out, (count,), (start + count,), tables.cuda(), 2)
        _check(out, expected, BF16, form)


@pytest.mark.parametrize("group,dim,page,count,start,window,bad", [case for case in NO_NUMBER if case[1] <= 128])
def test_what_is_no_number_stays_where_it_is_in_float(group, dim, page, count, start, window, bad):
    _no_number(F32, group, dim, page, count, start, window, bad)


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("dim,sink", [(64, False), (128, False), (64, True)])
def test_queries_that_see_nothing(kind, dim, sink):
    """Windows behind the table's end, pages that it does not have, a sink of minus infinity: zeros, as single tokens get them."""
    tables, pages, _, _ = _requests((1, 1), (79, 79), 16, 95)
    tables = tables[:, :5].contiguous()
    pools, _ = _cache(tables, pages, (80, 80), 2, dim, 16, 96)
    tables[1] = -1
    q = torch.randn((140, 2 * dim), generator=torch.Generator().manual_seed(97)).to(kind)
    sinks = torch.full((2,), -math.inf).cuda() if sink else None
    for form, run in _portions(kind, dim):
        out = torch.full((141, 2 * dim), -9.0, dtype=kind).cuda()
        run(q.cuda(), pools, out[:140], (70, 70), (160, 80), tables.cuda(), 2, 12, sinks)      # (at 90 .. and 10 ..)
        assert torch.equal(out[1:140], torch.zeros_like(out[1:140])), form
        assert bool((out[:1] != 0).any()) and bool((out[140] == -9.0).all()), form

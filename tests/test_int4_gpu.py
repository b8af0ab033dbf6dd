"""The cache in 4 bits on the GPU: what is written, what is read back, and attention over it, against plain formulas in
64 bits."""

import math

import numpy as np
import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _requests(counts, starts, page, seed, spare=3):
    """(tables [items, width] int32, pages, items and positions of all tokens): pages scattered, table entries that no
    request holds outside the pool."""
    g = torch.Generator().manual_seed(seed)
    needed = [-(-(start + count) // page) for count, start in zip(counts, starts)]
    pages = sum(needed) + spare
    order = torch.randperm(pages, generator=g).tolist()
    tables = torch.full((len(counts), max(needed) + 2), -1, dtype=torch.int32)
    tables[:, -1] = 1 << 30
    for item, count in enumerate(needed):
        tables[item, :count] = torch.tensor([order.pop() for _ in range(count)], dtype=torch.int32)
    items = [item for item, count in enumerate(counts) for _ in range(count)]
    positions = [start + j for count, start in zip(counts, starts) for j in range(count)]
    return tables, pages, items, positions


def _ints(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _garbage(pages, kv_heads, page, dim, seed):
    """A pool of bytes whose steps are NaN wherever nobody writes."""
    g = torch.Generator().manual_seed(seed)
    groups = -(-dim // 32)
    pool = torch.randint(0, 256, (pages, kv_heads, page, 18 * groups), dtype=torch.uint8, generator=g)
    pool.view(pages, kv_heads, -1)[:, :, page * 16 * groups:] = 0xff
    return pool


def _rows(n, kv_heads, dim, kind, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, kv_heads, dim), generator=g)
    x[..., 3::29] *= 5.0
    if n > 1 and dim > 1:
        x[n // 2, 0] = 0.0                                  # a group of zeros
        x[0, -1] = x[0, -1].abs().clamp(min=0.1).neg()      # all of one sign
        x[n - 1, 0, ::2] = -x[n - 1, 0, :dim - dim % 2:2].abs().max()    # the largest magnitude many times, both signs
        x[n - 1, 0, 1] = x[n - 1, 0].abs().max()
    return x.view(n, kv_heads * dim).to(kind)


def _tables_on(tables):
    return tables.cuda()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("kv_heads,dim,page,counts,starts", [
    (1, 1, 8, (1,), (0,)), (3, 16, 8, (5, 1, 9), (0, 7, 3)), (12, 64, 16, (1,) * 8, (0, 15, 16, 17, 40, 900, 3, 31)),
    (2, 48, 24, (30,), (11,)), (1, 33, 16, (17,), (5,)), (5, 96, 8, (3, 20), (100, 0)), (2, 128, 32, (40, 2), (0, 63)),
    (1, 256, 64, (70,), (60,)), (2, 250, 16, (7,), (0,))])
def test_written_and_read(kind, kv_heads, dim, page, counts, starts):
    """The bytes of every page and the values read back, exactly; nothing else in the pools changes."""
    from pagedserve_amd.ops import kernels

    tables, pages, items, positions = _requests(counts, starts, page, 1)
    tokens = len(items)
    wide = torch.zeros(tokens, 3 * kv_heads * dim + 1, dtype=kind)
    k, v = _rows(tokens, kv_heads, dim, kind, 2), _rows(tokens, kv_heads, dim, kind, 3)
    wide[:, 1:1 + kv_heads * dim] = k
    wide[:, -kv_heads * dim:] = v
    wide = wide.cuda()
    pools = [_garbage(pages, kv_heads, page, dim, seed) for seed in (4, 5)]
    on = [pool.cuda() for pool in pools]
    index = (_ints(items), _ints(positions), tables.cuda())
    kernels.kv_write_int4(wide[:, 1:1 + kv_heads * dim], wide[:, -kv_heads * dim:], *on, *index)
    read = [torch.full((tokens, kv_heads * dim), -3.0, dtype=kind).cuda() for _ in range(2)]
    kernels.kv_read_int4(*on, *read, *index)
    for keys, rows, pool, got, back in zip((True, False), (k, v), pools, on, read):
        codes, steps, values = plain.held(rows, kv_heads)
        plain.store(pool, codes, steps, tables.tolist(), items, positions, keys)
        assert torch.equal(got.cpu(), pool)
        assert torch.equal(back.double().cpu(), values)


def test_values_between_codes():
    """Floats on either side of the middle between two codes, which a rounded quotient cannot tell from it."""
    from pagedserve_amd.ops import kernels

    step = 0.8125
    rows = np.zeros((8, 32), dtype=np.float32)
    for t in range(8):
        middle = [np.float32((c + 0.5) * step) for c in range(-8, 7)]
        rows[t, :15] = middle
        rows[t, 15:30] = [np.nextafter(x, np.float32(9 if t % 2 else -9)) for x in middle]
        rows[t, 30] = -8 * step if t < 4 else 8 * step
        rows[t] *= np.float32(2.0) ** (t * 5 - 20)
    rows = torch.from_numpy(rows)
    tables, pages, items, positions = _requests((8,), (0,), 8, 6)
    pool = torch.zeros(pages, 1, 8, 18, dtype=torch.uint8).cuda()
    other = pool.clone()
    index = (_ints(items), _ints(positions), tables.cuda())
    kernels.kv_write_int4(rows.cuda(), rows.cuda(), pool, other, *index)
    back = [torch.zeros(8, 32).cuda() for _ in range(2)]
    kernels.kv_read_int4(pool, other, *back, *index)
    _, steps, values = plain.held(rows, 1)
    assert set(np.abs(np.ldexp(steps[:, 0, 0], [20 - 5 * t for t in range(8)]))) == {step}
    assert torch.equal(back[0].double().cpu(), values) and torch.equal(back[1].double().cpu(), values)


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("splits", [1, 64])
def test_positions_outside_the_table(kind, splits):
    """Positions far in front of the context are in front of it; one behind the table sees all that the table has."""
    from pagedserve_amd.ops import kernels

    tables, pages, _, _ = _requests((1, 1, 1), (49, 49, 49), 16, 12)
    tables = tables[:, :4].contiguous()
    pools, kept = _cache(tables, pages, (64, 64, 64), 2, 64, 16, 13)
    q = torch.randn((3, 128), generator=torch.Generator().manual_seed(14)).to(kind)
    out = torch.full((3, 128), 5.0, dtype=kind).cuda()
    kernels.attention_decode_int4(q.cuda(), *pools, out, None, _ints([-(1 << 31), (1 << 31) - 1, -64]), tables.cuda(), 2,
                                  0.125, splits, torch.zeros(3 * 2 * splits * 66).cuda())
    assert bool((out[0] == 0).all()) and bool((out[2] == 0).all())
    expected = list(plain.attention(q[1:2], *kept[1], [63], 2, 0.125))
    assert bool(((out[1:2].double().cpu() - expected[0]).abs() <= plain.allowed(*expected, kind, kind == BF16)).all())


@pytest.mark.parametrize("dim,size,ranges", [(64, 64, 1), (64, 128, 2), (128, 128, 1), (128, 64, 3), (256, 64, 1)])
def test_portions_that_pass_the_table(dim, size, ranges):
    """A portion whose last queries lie behind the block table: they see all that the table has, those in front as ever."""
    from pagedserve_amd.ops import kernels

    tables, pages, _, _ = _requests((1,), (111,), 16, 15)
    tables = tables[:, :7].contiguous()                        # 112 keys
    pools, kept = _cache(tables, pages, (112,), 1, dim, 16, 16)
    q = torch.randn((100, dim), generator=torch.Generator().manual_seed(17)).to(BF16)
    positions = list(range(50, 150))
    tiles = list(range(0, 100, size))
    out = torch.zeros((100, dim), dtype=BF16).cuda()
    kernels.attention_prefill_int4(q.cuda(), *pools, out, _ints([0] * len(tiles)), _ints(tiles), _ints([0, 100]),
                                   _ints([150]), tables.cuda(), 1, dim ** -0.5, query_tile=size, ranges=ranges)
    expected = list(plain.attention(q, *kept[0], [min(p, 111) for p in positions], 1, dim ** -0.5))
    assert bool(((out.double().cpu() - expected[0]).abs() <= plain.allowed(*expected, BF16, True)).all())


@pytest.mark.parametrize("kind", [BF16, F32])
def test_values_of_every_magnitude(kind):
    """Numbers of 8 bits, whose quotients by a step of 5 often are half way between two codes, from the smallest steps
    to the largest: the very codes of the definition."""
    from pagedserve_amd.ops import kernels

    g = torch.Generator().manual_seed(10)
    rows = torch.randint(-255, 256, (256, 128), generator=g).double()
    rows[::3] = torch.randint(-16, 17, (86, 128), generator=g).double() * 8 + 0.0
    for t in range(256):
        rows[t, 32 * (t % 4):32 * (t % 4) + 32] *= 0.125 ** (t % 3)
        rows[t] *= 2.0 ** (t - 136)                          # (the steps' exponents: -126 and below to 124)
    rows = rows.to(torch.float32).to(kind)
    tables, pages, items, positions = _requests((256,), (0,), 16, 11)
    pools = [torch.zeros(pages, 2, 16, 36, dtype=torch.uint8).cuda() for _ in range(2)]
    index = (_ints(items), _ints(positions), tables.cuda())
    kernels.kv_write_int4(rows.cuda(), rows.cuda(), *pools, *index)
    back = [torch.zeros(256, 128).cuda() for _ in range(2)]
    kernels.kv_read_int4(*pools, *back, *index)
    _, _, values = plain.held(rows, 2)
    for got in back:
        torch.testing.assert_close(got.double().cpu(), values, rtol=0, atol=0, equal_nan=True)


def test_values_that_are_no_numbers():
    """A group with a NaN or an infinity in it is NaN, its neighbours are not; tiny groups are zeros; tokens without a page
    are neither stored nor read."""
    from pagedserve_amd.ops import kernels

    rows = _rows(6, 2, 64, F32, 7)
    rows[0, 3] = math.nan
    rows[1, 40] = math.inf
    rows[2, 127] = -math.inf
    rows[3, :32] = 1e-38
    rows[3, 0] = 3e-38
    rows[4, 64:] = 3.4e38
    tables, pages, _, _ = _requests((6,), (0,), 8, 8)
    items, positions = [0] * 6, [0, 1, 2, 3, 4, 8 * (tables.shape[1] - 1)]
    pools = [torch.zeros(pages, 2, 8, 36, dtype=torch.uint8).cuda() for _ in range(2)]
    index = (_ints(items), _ints(positions), tables.cuda())
    kernels.kv_write_int4(rows.cuda(), rows.cuda(), *pools, *index)
    back = [torch.full((6, 128), 77.0).cuda() for _ in range(2)]
    kernels.kv_read_int4(*pools, *back, *index)
    _, _, values = plain.held(rows, 2)
    values[5] = 77.0
    for got in back:
        torch.testing.assert_close(got.double().cpu(), values, rtol=0, atol=0, equal_nan=True)
    assert bool(values[3, :32].eq(0).all()) and int(values.isnan().sum()) == 96


def _cache(tables, pages, lengths, kv_heads, dim, page, seed):
    """Pools that hold every request's keys and values, NaN elsewhere, and those keys and values per request."""
    pools = [_garbage(pages, kv_heads, page, dim, seed + which) for which in range(2)]
    kept = []
    for item, length in enumerate(lengths):
        pair = []
        for which, keys in enumerate((True, False)):
            codes, steps, values = plain.held(_rows(length, kv_heads, dim, F32, seed + 10 * item + which), kv_heads)
            plain.store(pools[which], codes, steps, tables.tolist(), [item] * length, list(range(length)), keys)
            pair.append(values)
        kept.append(pair)
    return [pool.cuda() for pool in pools], kept


DECODE = [
    # kv_heads, group, dim, page, lengths, window, sink, softcap
    (1, 1, 64, 8, (1,), 0, False, 0.0), (12, 1, 64, 16, (1, 2, 15, 16, 17, 130), 0, False, 0.0),
    (2, 8, 128, 16, (33, 300, 7), 0, False, 0.0), (1, 16, 128, 32, (65, 64, 1), 0, True, 0.0),
    (4, 4, 16, 8, (19, 100), 0, False, 20.0), (5, 3, 48, 24, (25, 71, 90), 0, True, 0.0),
    (2, 2, 96, 16, (40, 129), 33, False, 0.0), (2, 1, 256, 64, (70, 200), 0, True, 15.0),
    (3, 1, 32, 8, (60, 9), -16, False, 0.0), (2, 3, 80, 16, (50, 31), 7, True, 0.0),
    (1, 2, 250, 16, (20,), 0, False, 0.0), (2, 1, 1, 8, (9, 30), 0, False, 0.0), (1, 5, 7, 8, (40,), -8, False, 0.0),
    (1, 20, 64, 16, (90, 3), 0, False, 0.0), (2, 40, 128, 8, (50,), 20, True, 0.0)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("kv_heads,group,dim,page,lengths,window,sink,softcap", DECODE)
def test_single_tokens(kind, kv_heads, group, dim, page, lengths, window, sink, softcap):
    """One query a request, in one range and in several, with and without a list of tokens; rows behind stay as they were."""
    from pagedserve_amd.ops import kernels

    heads = kv_heads * group
    tables, pages, _, _ = _requests([1] * len(lengths), [length - 1 for length in lengths], page, 21)
    pools, kept = _cache(tables, pages, lengths, kv_heads, dim, page, 22)
    g = torch.Generator().manual_seed(23)
    n = len(lengths)
    q = (torch.randn((n, heads * dim), generator=g) * 1.5).to(kind)
    sinks = torch.randn(heads, generator=g).cuda() if sink else None
    scale = dim ** -0.5
    expected = [list(plain.attention(q[i:i + 1], *kept[i], [length - 1], heads, scale, window, sinks, softcap))
                for i, length in enumerate(lengths)]
    expected = [torch.cat([e[which] for e in expected]) for which in range(3)]
    limit = plain.allowed(*expected, kind, kind == BF16)
    positions = _ints([length - 1 for length in lengths])
    picked = list(range(n))[::-1][:max(1, n - 1)]
    for splits in (1, 2, 5):
        partial = torch.full((n * heads * splits * (dim + 2),), math.nan).cuda() if splits > 1 else None
        out = torch.full((n + 1, heads * dim), -9.0, dtype=kind).cuda()
        kernels.attention_decode_int4(q.cuda(), *pools, out[:n], None, positions, tables.cuda(), heads, scale, splits,
                                      partial, window, sink=sinks, softcap=softcap)
        assert bool(((out[:n].double().cpu() - expected[0]).abs() <= limit).all()), splits
        assert bool((out[n] == -9.0).all())
        out.fill_(-9.0)
        kernels.attention_decode_int4(q.cuda(), *pools, out[:n], _ints(list(range(n))), positions, tables.cuda(), heads,
                                      scale, splits, partial, window, tok_list=_ints(picked), sink=sinks, softcap=softcap)
        off = (out[:n].double().cpu() - expected[0]).abs() <= limit
        assert bool(off[picked].all())
        rest = [i for i in range(n + 1) if i not in picked]
        assert bool((out[rest] == -9.0).all())


@pytest.mark.parametrize("kind", [F32, BF16])
def test_tokens_that_see_nothing(kind):
    """A position in front of the context, and pages outside the pool, give zeros; a NaN behind a query does not reach it."""
    from pagedserve_amd.ops import kernels

    tables, pages, _, _ = _requests((1, 1, 1), (19, 19, 39), 8, 31)
    pools, kept = _cache(tables, pages, (20, 20, 40), 2, 64, 8, 32)
    q = torch.randn((3, 128), generator=torch.Generator().manual_seed(33)).to(kind)
    missing = tables.clone()
    missing[1] = 1 << 29
    positions = [-1, 19, 20]
    for window in (0, -8, 5):
        for splits in (1, 3):
            out = torch.full((3, 128), 5.0, dtype=kind).cuda()
            partial = torch.zeros(3 * 2 * splits * 66).cuda()
            kernels.attention_decode_int4(q.cuda(), *pools, out, None, _ints(positions), missing.cuda(), 2, 0.125, splits,
                                          partial, window)
            assert bool((out[:2] == 0).all())
            out_1, size, shift = plain.attention(q[2:], kept[2][0][:21], kept[2][1][:21], [20], 2, 0.125, window)
            assert bool(((out[2:].double().cpu() - out_1).abs() <= plain.allowed(out_1, size, shift, kind, kind == BF16)).all())


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("splits", [1, 2])
def test_sinks_of_minus_infinity(kind, splits):
    """A sink that weighs nothing: attention without one, and zeros for a token that sees nothing."""
    from pagedserve_amd.ops import kernels

    tables, pages, _, _ = _requests((1, 1), (19, 299), 16, 34)
    pools, kept = _cache(tables, pages, (20, 300), 2, 64, 16, 35)
    q = torch.randn((2, 128), generator=torch.Generator().manual_seed(36)).to(kind)
    sinks = torch.tensor([-math.inf, 0.5]).cuda()
    out = torch.full((2, 128), 5.0, dtype=kind).cuda()
    kernels.attention_decode_int4(q.cuda(), *pools, out, None, _ints([-1, 299]), tables.cuda(), 2, 0.125, splits,
                                  torch.zeros(2 * 2 * splits * 66).cuda(), sink=sinks)
    assert bool((out[0] == 0).all())
    expected = list(plain.attention(q[1:], *kept[1], [299], 2, 0.125, 0, sinks))
    assert bool(((out[1:].double().cpu() - expected[0]).abs() <= plain.allowed(*expected, kind, kind == BF16)).all())


STORED = [
    # kv_heads, group, dim, page, lengths (the stored key among them), window, splits
    (3, 1, 64, 16, (1, 32, 33, 200, 129), 0, 1), (2, 8, 128, 32, (700, 64, 5, 128), 0, 4), (1, 4, 32, 8, (90, 8, 9), 40, 2),
    (2, 2, 96, 24, (50, 500), 0, 3), (1, 1, 256, 16, (300, 1), -64, 1), (2, 1, 33, 40, (41, 40, 260), 0, 8),
    (1, 20, 64, 16, (140, 77), 0, 2), (1, 2, 160, 8, (66,), 0, 1), (1, 12, 192, 16, (150, 31), 0, 2), (2, 1, 7, 16, (17, 400), 0, 5),
    (1, 1, 224, 64, (64, 65), 0, 1)]


@pytest.mark.parametrize("kv_heads,group,dim,page,lengths,window,splits", STORED)
def test_tokens_that_store_their_own_rows(kv_heads, group, dim, page, lengths, window, splits):
    """One launch does what storing and attending do, bit for bit, in the pools too; a token in front of its context, one
    behind the table and one whose page does not exist store nothing."""
    from pagedserve_amd.ops import kernels

    heads, items = kv_heads * group, len(lengths) + 3
    tables, pages, _, _ = _requests((*lengths, 20, 20, 20), (0,) * items, page, 71)
    pools, _ = _cache(tables, pages, [max(1, length - 1) for length in lengths] + [20, 20, 19], kv_heads, dim, page, 72)
    tables[-1, 19 // page] = -1
    g = torch.Generator().manual_seed(73)
    both = torch.randn((items, (heads + 2 * kv_heads) * dim + 3), generator=g).to(BF16)
    both[0, heads * dim + 2] = 1e4                           # (a step far above the others)
    both = both.cuda()
    q, k, v = both[:, :-3].split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    positions = _ints([length - 1 for length in lengths] + [-1, tables.shape[1] * page + 3, 19])
    results = []
    for together in (False, True):
        mine = [pool.clone() for pool in pools]
        out = torch.full((items, heads * dim), 7.0, dtype=BF16).cuda()
        partial = torch.full((items * heads * splits * (dim + 2),), math.nan).cuda()
        if not together:
            kernels.kv_write_int4(k, v, *mine, _ints(list(range(items))), positions, tables.cuda())
        kernels.attention_decode_int4(q, *mine, out, None, positions, tables.cuda(), heads, dim ** -0.5, splits, partial, window,
                                      store=(k, v) if together else None)
        results.append((out, *mine))
    # (the token behind the table sees places that nobody filled)
    torch.testing.assert_close(results[1][0], results[0][0], rtol=0, atol=0, equal_nan=True)
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])
    assert bool((results[1][0][-3] == 0).all()) and not bool(results[1][0][:-2].isnan().any() or results[1][0][-1].isnan().any())


@pytest.mark.parametrize("kind", [BF16, F32])
@pytest.mark.parametrize("size", [1e9, 1e25])
def test_scores_of_any_size(kind, size):
    """Keys so large that the best score alone counts: its value, whatever the score's rounding."""
    from pagedserve_amd.ops import kernels

    tables, pages, items, positions = _requests((90,), (0,), 16, 77)
    pools = [_garbage(pages, 1, 16, 64, 78 + which) for which in range(2)]
    pools = [pool.cuda() for pool in pools]
    g = torch.Generator().manual_seed(79)
    k = torch.randn((90, 64), generator=g)
    k[:, 0] = torch.randperm(90, generator=g) - 45.0
    k[17, 0], k[71, 0] = 90.0, -90.0                         # (the scores' ends)
    v = torch.randn((90, 64), generator=g)
    kernels.kv_write_int4((k * size).cuda(), v.cuda(), *pools, _ints(items), _ints(positions), tables.cuda())
    kept = [torch.zeros(90, 64).cuda() for _ in range(2)]
    kernels.kv_read_int4(*pools, *kept, _ints(items), _ints(positions), tables.cuda())
    q = torch.zeros(2, 64)
    q[0, 0], q[1, 0] = 3.0, -3.0
    best = [17, 71]
    for splits in (1, 2):
        out = torch.zeros(2, 64, dtype=kind).cuda()
        kernels.attention_decode_int4(q.to(kind).cuda(), *pools, out, _ints([0, 0]), _ints([89, 89]), tables.cuda(), 1, 0.125,
                                      splits, torch.zeros(2 * splits * 66).cuda())
        expected = kept[1][best]
        assert bool(((out.float() - expected).abs() <= 2.0 ** -7 * expected.abs().amax(1, keepdim=True)).all())
    tiles = (_ints([0]), _ints([0]), _ints([0, 2]), _ints([90]), tables.cuda(), 1, 0.125)
    q = q.to(kind).cuda()                                    # (positions 88 and 89, behind both ends)
    out = torch.zeros(2, 64, dtype=kind).cuda()
    if kind == F32:
        kernels.attention_tiled_f32_int4(q, *pools, out, *tiles)
        assert bool(((out - expected).abs() <= 2.0 ** -7 * expected.abs().amax(1, keepdim=True)).all())
    else:
        for query_tile, ranges in ((64, 1), (128, 1), (64, 2)):
            kernels.attention_prefill_int4(q, *pools, out, *tiles, query_tile=query_tile, ranges=ranges)
            assert bool(((out.float() - expected).abs() <= 2.0 ** -7 * expected.abs().amax(1, keepdim=True)).all())


def test_a_stored_row_that_is_no_number():
    """A NaN in the token's own value makes its group's result one, a NaN in its key the head's, and nothing else."""
    from pagedserve_amd.ops import kernels

    tables, pages, _, _ = _requests((40, 40, 40), (0, 0, 0), 16, 74)
    pools, _ = _cache(tables, pages, (39, 39, 39), 2, 64, 16, 75)
    rows = torch.randn((3, 384), generator=torch.Generator().manual_seed(76)).to(BF16).cuda()
    rows[1, 128 + 3] = math.nan                              # a key's first head
    rows[2, 256 + 64 + 40] = math.inf                        # a value's second head, second group
    out = torch.zeros(3, 128, dtype=BF16).cuda()
    kernels.attention_decode_int4(rows[:, :128], *pools, out, None, _ints([39, 39, 39]), tables.cuda(), 2, 0.125, 1,
                                  store=(rows[:, 128:256], rows[:, 256:]))
    bad = out.isnan().cpu()
    assert not bad[0].any() and bad[1, :64].all() and not bad[1, 64:].any()
    assert bad[2, 96:].all() and not bad[2, :96].any()


PROMPT = [
    # kv_heads, group, dim, page, counts, starts, window, sink, softcap
    (1, 1, 64, 8, (2,), (0,), 0, False, 0.0), (3, 1, 64, 16, (65, 130), (0, 0), 0, False, 0.0),
    (2, 4, 128, 16, (33, 70, 2), (100, 0, 31), 0, False, 0.0), (1, 2, 16, 8, (40,), (3,), 0, True, 0.0),
    (2, 1, 48, 24, (100, 20), (0, 50), 0, False, 30.0), (1, 3, 96, 16, (64,), (10,), 40, False, 0.0),
    (1, 1, 256, 64, (70,), (20,), 0, True, 0.0), (1, 2, 80, 8, (35,), (5,), -16, False, 0.0), (2, 6, 112, 16, (70, 9), (40, 0), 30, True, 20.0),
    (1, 2, 128, 8, (64, 65, 1, 40), (0, 7, 130, 9), 0, True, 0.0),
    (1, 1, 160, 16, (50,), (0,), 0, False, 0.0), (2, 1, 32, 8, (129,), (200,), 0, False, 0.0), (1, 1, 112, 8, (60,), (8,), 0, False, 0.0)]


@pytest.mark.parametrize("kv_heads,group,dim,page,counts,starts,window,sink,softcap", PROMPT)
def test_prompt_portions(kv_heads, group, dim, page, counts, starts, window, sink, softcap):
    """Whole prompts and later portions in every size of tile that takes the head size, and token by token."""
    from pagedserve_amd.ops import kernels

    heads = kv_heads * group
    tables, pages, items, positions = _requests(counts, starts, page, 41)
    lengths = [a + b for a, b in zip(counts, starts)]
    pools, kept = _cache(tables, pages, lengths, kv_heads, dim, page, 42)
    tokens = sum(counts)
    g = torch.Generator().manual_seed(43)
    q = (torch.randn((tokens, heads * dim), generator=g) * 1.5).to(BF16)
    sinks = torch.randn(heads, generator=g).cuda() if sink else None
    scale = dim ** -0.5
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    parts = [list(plain.attention(q[cu[i]:cu[i + 1]], *kept[i], positions[cu[i]:cu[i + 1]], heads, scale, window, sinks,
                                  softcap)) for i in range(len(counts))]
    expected = [torch.cat([part[which] for part in parts]) for which in range(3)]
    limit = plain.allowed(*expected, BF16, True)
    for size in (64, 128):
        if size == 128 and dim > 128:
            continue
        tiles = [(item, q0) for item, count in enumerate(counts) for q0 in range(0, count, size)]
        pairs = size == 64 < dim <= 128 and group % 2 == 0
        for max_kv_len, ranges, pair in ((100, None, None), (0, 1, 1), (600, 1, 1), (0, 2, 1), (600, 5, 1),
                                         *([(0, 1, 2), (600, 3, 2)] if pairs else [])):      # (they steer the launch)
            out = torch.full((tokens + 1, heads * dim), -9.0, dtype=BF16).cuda()
            kernels.attention_prefill_int4(q.cuda(), *pools, out[:tokens], _ints([t[0] for t in tiles]),
                                           _ints([t[1] for t in tiles]), _ints(cu), _ints(lengths), tables.cuda(), heads,
                                           scale, window, max_kv_len, size, sinks, softcap, pair, ranges)
            assert bool(((out[:tokens].double().cpu() - expected[0]).abs() <= limit).all()), (size, max_kv_len, ranges, pair)
            assert bool((out[tokens] == -9.0).all())
    out = torch.zeros((tokens, heads * dim), dtype=BF16).cuda()
    kernels.attention_decode_int4(q.cuda(), *pools, out, _ints(items), _ints(positions), tables.cuda(), heads, scale, 1,
                                  None, window, sink=sinks, softcap=softcap)
    assert bool(((out.double().cpu() - expected[0]).abs() <= limit).all())


FLOAT = [
    # kv_heads, group, dim, page, counts, starts, window, sink, softcap
    (3, 1, 64, 16, (65, 130), (0, 0), 0, False, 0.0), (2, 4, 128, 16, (33, 70, 2), (100, 0, 31), 0, False, 0.0),
    (1, 2, 16, 8, (40,), (3,), 0, True, 0.0), (2, 1, 48, 24, (100, 20), (0, 50), 0, False, 30.0),
    (1, 3, 96, 16, (64,), (10,), 40, False, 0.0), (1, 2, 80, 8, (35,), (5,), -16, False, 0.0), (1, 2, 20, 8, (50, 3), (0, 61), 0, False, 0.0),
    (2, 1, 32, 8, (129,), (200,), 0, True, 0.0), (1, 1, 124, 40, (60,), (8,), 25, False, 20.0), (1, 1, 4, 8, (33,), (1,), 0, False, 0.0)]


@pytest.mark.parametrize("kv_heads,group,dim,page,counts,starts,window,sink,softcap", FLOAT)
def test_prompt_portions_in_float(kv_heads, group, dim, page, counts, starts, window, sink, softcap):
    """Float queries, in every form of tile; the row behind the last token stays."""
    from pagedserve_amd.ops import kernels

    heads = kv_heads * group
    tables, pages, _, positions = _requests(counts, starts, page, 47)
    lengths = [a + b for a, b in zip(counts, starts)]
    pools, kept = _cache(tables, pages, lengths, kv_heads, dim, page, 48)
    tokens = sum(counts)
    g = torch.Generator().manual_seed(49)
    q = torch.randn((tokens, heads * dim), generator=g) * 1.5
    sinks = torch.randn(heads, generator=g).cuda() if sink else None
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    parts = [list(plain.attention(q[cu[i]:cu[i + 1]], *kept[i], positions[cu[i]:cu[i + 1]], heads, dim ** -0.5, window, sinks,
                                  softcap)) for i in range(len(counts))]
    expected = [torch.cat([part[which] for part in parts]) for which in range(3)]
    limit = plain.allowed(*expected, F32, False)
    for size, paired in ((32, False), (64, False), (64, True)):
        tiles = [(item, q0) for item, count in enumerate(counts) for q0 in range(0, count, size)]
        out = torch.full((tokens + 1, heads * dim), -9.0).cuda()
        kernels.attention_tiled_f32_int4(q.cuda(), *pools, out[:tokens], _ints([t[0] for t in tiles]),
                                         _ints([t[1] for t in tiles]), _ints(cu), _ints(lengths), tables.cuda(), heads,
                                         dim ** -0.5, window, sinks, softcap, size, paired)
        assert bool(((out[:tokens].double().cpu() - expected[0]).abs() <= limit).all()), (size, paired)
        assert bool((out[tokens] == -9.0).all())


@pytest.mark.parametrize("bad", ["key", "value"])
def test_a_later_nan_reaches_no_earlier_float_query(bad):
    from pagedserve_amd.ops import kernels

    tables, pages, _, positions = _requests((40,), (100,), 8, 54)
    (k_pool, v_pool), kept = _cache(tables, pages, (140,), 1, 64, 8, 55)
    rows = [torch.zeros(2, 64), torch.zeros(2, 64)]
    rows[bad == "value"][:, 5] = math.nan
    kernels.kv_write_int4(rows[0].cuda(), rows[1].cuda(), k_pool, v_pool, _ints([0, 0]), _ints([139, 110]), tables.cuda())
    q = torch.randn((40, 64), generator=torch.Generator().manual_seed(56))
    expected = list(plain.attention(q[:10], kept[0][0][:110], kept[0][1][:110], positions[:10], 1, 0.125))
    for size, paired in ((32, False), (64, False), (64, True)):
        tiles = list(range(0, 40, size))
        out = torch.zeros(40, 64).cuda()
        kernels.attention_tiled_f32_int4(q.cuda(), k_pool, v_pool, out, _ints([0] * len(tiles)), _ints(tiles), _ints([0, 40]),
                                         _ints([140]), tables.cuda(), 1, 0.125, query_tile=size, paired=paired)
        assert bool(((out[:10].double().cpu() - expected[0]).abs() <= plain.allowed(*expected, F32, False)).all())
        assert bool(out[10:].isnan().any(1).all())


LONG = [
    # kv_heads, group, dim, page, counts, starts, window, sink, softcap, query_tile
    (2, 2, 64, 16, (70, 3), (1500, 40), 0, True, 0.0, 64), (1, 4, 64, 24, (130,), (900,), 300, False, 0.0, 128),
    (1, 2, 128, 8, (20, 64), (1100, 700), 0, False, 20.0, 64), (1, 1, 128, 16, (140,), (1000,), 0, True, 0.0, 128), (1, 1, 256, 16, (66,), (800,), -256, True, 0.0, 64)]


@pytest.mark.parametrize("kv_heads,group,dim,page,counts,starts,window,sink,softcap,size", LONG)
def test_prompt_portions_in_ranges(kv_heads, group, dim, page, counts, starts, window, sink, softcap, size):
    """Ranges of keys of long contexts, as the rule cuts them and in numbers that leave some without keys; the scratch holds
    what is no number before, and what lies behind its records stays."""
    from pagedserve_amd.ops import kernels

    heads = kv_heads * group
    tables, pages, _, positions = _requests(counts, starts, page, 44)
    lengths = [a + b for a, b in zip(counts, starts)]
    pools, kept = _cache(tables, pages, lengths, kv_heads, dim, page, 45)
    tokens = sum(counts)
    g = torch.Generator().manual_seed(46)
    q = (torch.randn((tokens, heads * dim), generator=g) * 1.5).to(BF16)
    sinks = torch.randn(heads, generator=g).cuda() if sink else None
    scale = dim ** -0.5
    cu = [sum(counts[:i]) for i in range(len(counts) + 1)]
    parts = [list(plain.attention(q[cu[i]:cu[i + 1]], *kept[i], positions[cu[i]:cu[i + 1]], heads, scale, window, sinks,
                                  softcap)) for i in range(len(counts))]
    expected = [torch.cat([part[which] for part in parts]) for which in range(3)]
    limit = plain.allowed(*expected, BF16, True)
    tiles = [(item, q0) for item, count in enumerate(counts) for q0 in range(0, count, size)]
    rule = kernels.prefill_int4_ranges(len(tiles), heads, max(lengths))
    assert rule > 1
    for ranges, pair in ((rule, 1), (7, 1), (64, 1), *([(rule, 2), (5, 2)] if dim == 128 and group == 2 else [])):
        needed = len(tiles) * heads * ranges * size * (dim + 2)
        partial = torch.full((needed + 8,), math.nan).cuda()
        out = torch.full((tokens + 1, heads * dim), -9.0, dtype=BF16).cuda()
        kernels.attention_prefill_int4(q.cuda(), *pools, out[:tokens], _ints([t[0] for t in tiles]),
                                       _ints([t[1] for t in tiles]), _ints(cu), _ints(lengths), tables.cuda(), heads, scale,
                                       window, max(lengths), size, sinks, softcap, pair, ranges, partial)
        assert bool(((out[:tokens].double().cpu() - expected[0]).abs() <= limit).all()), (ranges, pair)
        assert bool((out[tokens] == -9.0).all()) and bool(partial[needed:].isnan().all())
    with pytest.raises(kernels.KernelError, match="floats of scratch"):
        kernels.attention_prefill_int4(q.cuda(), *pools, out[:tokens], _ints([t[0] for t in tiles]),
                                       _ints([t[1] for t in tiles]), _ints(cu), _ints(lengths), tables.cuda(), heads, scale,
                                       window, max(lengths), size, sinks, softcap, pair, ranges, partial[:-9])


@pytest.mark.parametrize("bad", ["key", "value"])
def test_a_later_nan_reaches_no_earlier_query(bad):
    """The last key (or value) of a portion is no number: the queries in front of it do not see it, the last one does."""
    from pagedserve_amd.ops import kernels

    tables, pages, items, positions = _requests((40,), (0,), 8, 51)
    (k_pool, v_pool), kept = _cache(tables, pages, (40,), 1, 64, 8, 52)
    rows = [torch.zeros(1, 64), torch.zeros(1, 64)]
    rows[bad == "value"][0, 5] = math.nan
    index = (_ints([0]), _ints([39]), tables.cuda())
    kernels.kv_write_int4(rows[0].cuda(), rows[1].cuda(), k_pool, v_pool, *index)
    q = torch.randn((40, 64), generator=torch.Generator().manual_seed(53)).to(BF16)
    expected = list(plain.attention(q[:39], kept[0][0][:39], kept[0][1][:39], positions[:39], 1, 0.125))
    for size, ranges in ((64, 1), (128, 1), (64, 3), (128, 2)):
        tiles = list(range(0, 40, size))
        out = torch.zeros(40, 64, dtype=BF16).cuda()
        kernels.attention_prefill_int4(q.cuda(), k_pool, v_pool, out, _ints([0] * len(tiles)), _ints(tiles), _ints([0, 40]),
                                       _ints([40]), tables.cuda(), 1, 0.125, query_tile=size, ranges=ranges)
        assert bool(((out[:39].double().cpu() - expected[0]).abs() <= plain.allowed(*expected, BF16, True)).all())
        assert bool(out[39].isnan().any())
    out = torch.zeros(40, 64, dtype=BF16).cuda()
    kernels.attention_decode_int4(q.cuda(), k_pool, v_pool, out, _ints(items), _ints(positions), tables.cuda(), 1, 0.125, 1)
    assert bool(((out[:39].double().cpu() - expected[0]).abs() <= plain.allowed(*expected, BF16, True)).all())
    assert bool(out[39].isnan().any())


def test_as_a_bfloat16_cache_of_the_values_held():
    """What a step would do, on the cache of the model's type holding the same values: the same attention."""
    from pagedserve_amd.ops import kernels

    heads, dim, page, counts = 4, 64, 16, (70, 1, 1)
    starts = (0, 200, 77)
    tables, pages, items, positions = _requests(counts, starts, page, 61)
    lengths = [a + b for a, b in zip(counts, starts)]
    pools, kept = _cache(tables, pages, lengths, heads, dim, page, 62)
    plain_pools = [torch.zeros(pages, heads, page, dim, dtype=BF16).cuda() for _ in range(2)]
    for item, length in enumerate(lengths):
        kernels.kv_write(*[x.to(BF16).cuda() for x in kept[item]], *plain_pools, _ints([item] * length),
                         _ints(list(range(length))), tables.cuda())
    q = torch.randn((72, heads * dim), generator=torch.Generator().manual_seed(63)).to(BF16).cuda()
    cu, tiles = _ints([0, 70, 71, 72]), (_ints([0, 0]), _ints([0, 64]))
    outs = []
    for four in (True, False):
        out = torch.zeros(72, heads * dim, dtype=BF16).cuda()
        prefill = kernels.attention_prefill_int4 if four else kernels.attention_prefill
        decode = kernels.attention_decode_int4 if four else kernels.attention_decode
        use = pools if four else plain_pools
        prefill(q, *use, out, *tiles, cu, _ints(lengths), tables.cuda(), heads, 0.125, max_kv_len=201)
        decode(q, *use, out, _ints(items), _ints(positions), tables.cuda(), heads, 0.125, 1, tok_list=_ints([70, 71]))
        outs.append(out.double().cpu())
    assert torch.equal(outs[0][:70], outs[1][:70])           # the same products in the same order
    expected = [list(plain.attention(q[t:t + 1], *kept[items[t]], [positions[t]], heads, 0.125)) for t in (70, 71)]
    for t, e in zip((70, 71), expected):
        limit = plain.allowed(*e, BF16, True)
        for out in outs:
            assert bool(((out[t:t + 1] - e[0]).abs() <= limit).all())


@pytest.mark.parametrize("dim,kv_heads,group,window,sink,softcap", [
    (16, 2, 1, 0, False, 0.0), (32, 1, 2, 0, True, 0.0), (48, 2, 3, 30, False, 0.0), (64, 1, 4, -16, False, 20.0),
    (128, 2, 1, 0, True, 0.0), (250, 1, 2, 0, False, 0.0)])
@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("kind", [BF16, F32])
def test_scales_that_are_not_positive(kind, scale, dim, kv_heads, group, window, sink, softcap):
    """Bfloat16 queries take another kernel under such a scale, a head to a block."""
    from pagedserve_amd.ops import kernels

    heads, lengths, page = kv_heads * group, (1, 17, 200, 530), 16
    tables, pages, _, _ = _requests([1] * len(lengths), [length - 1 for length in lengths], page, 101)
    pools, kept = _cache(tables, pages, lengths, kv_heads, dim, page, 102)
    q = torch.randn((len(lengths), heads * dim), generator=torch.Generator().manual_seed(103)).to(kind)
    sinks = torch.randn(heads, generator=torch.Generator().manual_seed(104)).cuda() if sink else None
    expected = [list(plain.attention(q[i:i + 1], *kept[i], [length - 1], heads, scale, window, sinks, softcap))
                for i, length in enumerate(lengths)]
    expected = [torch.cat([e[which] for e in expected]) for which in range(3)]
    limit = plain.allowed(*expected, kind, False)
    for splits in (1, 3):
        out = torch.full((len(lengths), heads * dim), -9.0, dtype=kind).cuda()
        kernels.attention_decode_int4(q.cuda(), *pools, out, None, _ints([length - 1 for length in lengths]), tables.cuda(), heads,
                                      scale, splits, torch.full((len(lengths) * heads * splits * (dim + 2),), math.nan).cuda(),
                                      window, sink=sinks, softcap=softcap)
        assert bool(((out.double().cpu() - expected[0]).abs() <= limit).all()), splits

"""The operators of the cache in 4 bits and the log probabilities as a serving program runs them: one after the other,
captured into graphs that share their scratch, on another stream, and over addresses beyond 32 bits."""

import math

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


class Step:
    """A step of three requests over a cache in 4 bits: a portion of 70 tokens behind 600 and single tokens behind 500 and
    39, whose rows go on to logits and log probabilities.  Buffers are made once, as a program that captures does."""

    HEADS, KV, DIM, PAGE, VOCAB = 8, 4, 64, 16, 9000
    COUNTS, STARTS = (70, 1, 1), (600, 500, 39)

    def __init__(self, scratch, seed):
        from pagedserve_amd.ops import kernels

        g = torch.Generator().manual_seed(seed)
        tokens = sum(self.COUNTS)
        lengths = [a + b for a, b in zip(self.COUNTS, self.STARTS)]
        needed = [-(-length // self.PAGE) for length in lengths]
        order = torch.randperm(sum(needed), generator=g).int()
        tables = torch.full((3, max(needed)), -1, dtype=torch.int32)
        for i, count in enumerate(needed):
            tables[i, :count] = order[sum(needed[:i]):sum(needed[:i + 1])]
        ints = lambda values: torch.tensor(values, dtype=torch.int32).cuda()
        self.kernels, self.tokens, self.lengths, self.scratch = kernels, tokens, lengths, scratch
        self.tables = tables.cuda()
        shape = (sum(needed), self.KV, self.PAGE, kernels.int4_row_bytes(self.DIM))
        self.pools = [torch.zeros(shape, dtype=torch.uint8).cuda() for _ in range(2)]
        # every key in front of the step
        items = [i for i, start in enumerate(self.STARTS) for _ in range(start)]
        positions = [p for start in self.STARTS for p in range(start)]
        before = [torch.randn(len(items), self.KV * self.DIM, generator=g).to(BF16) for _ in range(2)]
        kernels.kv_write_int4(*[x.cuda() for x in before], *self.pools, ints(items), ints(positions), self.tables)
        self.items = ints([i for i, count in enumerate(self.COUNTS) for _ in range(count)])
        self.positions = ints([s + j for c, s in zip(self.COUNTS, self.STARTS) for j in range(c)])
        self.cu, self.kv_lens = ints([0, 70, 71, 72]), ints(lengths)
        self.tile_item, self.tile_q0, self.singles = ints([0, 0]), ints([0, 64]), ints([70, 71])
        width = (self.HEADS + 2 * self.KV) * self.DIM
        self.qkv = torch.zeros(tokens, width, dtype=BF16).cuda()
        self.context = torch.zeros(tokens, self.HEADS * self.DIM, dtype=BF16).cuda()
        self.head = (torch.randn(self.VOCAB, self.HEADS * self.DIM, generator=g) * 0.3).to(BF16).cuda()
        self.logits = torch.zeros(tokens, self.VOCAB).cuda()
        self.wanted = torch.randint(0, self.VOCAB, (tokens,), generator=g).int().cuda()
        self.scores, self.entropy = torch.zeros(tokens).cuda(), torch.zeros(tokens).cuda()
        self.ids, self.best = ints([[0] * 5] * tokens), torch.zeros(tokens, 5).cuda()

    def results(self):
        return [self.context, self.logits, self.scores, self.entropy, self.ids, self.best, *self.pools]

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed)
        self.qkv.copy_((torch.randn(self.qkv.shape, generator=g) * 1.3).to(BF16))

    def clear(self):
        for x in self.results()[:6]:
            x.zero_()

    def run(self):
        kernels, columns = self.kernels, self.HEADS * self.DIM
        q, k, v = self.qkv.split([columns, self.KV * self.DIM, self.KV * self.DIM], 1)
        kernels.kv_write_int4(k, v, *self.pools, self.items, self.positions, self.tables)
        kernels.attention_decode_int4(q, *self.pools, self.context, self.items, self.positions, self.tables, self.HEADS,
                                      self.DIM ** -0.5, 4, self.scratch, tok_list=self.singles)
        kernels.attention_prefill_int4(q, *self.pools, self.context, self.tile_item, self.tile_q0, self.cu, self.kv_lens,
                                       self.tables, self.HEADS, self.DIM ** -0.5, max_kv_len=max(self.lengths), ranges=3,
                                       partial=self.scratch)
        kernels.linear(self.context, self.head, None, self.logits)
        kernels.token_logprobs(self.logits, self.wanted, self.scores, self.entropy, None, self.ids, self.best, self.scratch)


def _scratch():
    return torch.full((2 * 8 * 3 * 64 * 66,), math.nan).cuda()


def test_a_step_against_its_formulas():
    """Written, attended and scored one after the other: every stage against 64 bits, from what the stage before left."""
    step = Step(_scratch(), 1)
    step.fill(2)
    step.run()
    columns = step.HEADS * step.DIM
    q = step.qkv[:, :columns].cpu()
    for item, (count, start) in enumerate(zip(step.COUNTS, step.STARTS)):
        length, first = count + start, sum(step.COUNTS[:item])
        index = (torch.full((length,), item, dtype=torch.int32).cuda(), torch.arange(length, dtype=torch.int32).cuda())
        keys, values = [torch.zeros(length, step.KV * step.DIM).cuda() for _ in range(2)]
        step.kernels.kv_read_int4(*step.pools, keys, values, *index, step.tables)
        rows = step.qkv[first:first + count].cpu().float()
        assert torch.equal(keys[start:].double().cpu(), plain.held(rows[:, columns:columns + 256], step.KV)[2])
        assert torch.equal(values[start:].double().cpu(), plain.held(rows[:, columns + 256:], step.KV)[2])
        expected = list(plain.attention(q[first:first + count], keys.double().cpu(), values.double().cpu(),
                                        list(range(start, length)), step.HEADS, step.DIM ** -0.5))
        got = step.context[first:first + count].double().cpu()
        assert bool(((got - expected[0]).abs() <= plain.allowed(*expected, BF16, True)).all()), item
    chosen, entropy, _, ids, best = plain.logprobs(step.logits.cpu(), step.wanted.cpu(), 5)
    # (a logit is one float, the logarithm of a sum of exponentials of them a few roundings of numbers up to |logit| + 10)
    limit = 2.0 ** -24 * 32 * (step.logits.abs().max().item() + 10)
    assert bool(((step.scores.double().cpu() - chosen).abs() <= limit).all())
    assert bool(((step.best.double().cpu() - best).abs() <= limit).all())
    assert bool(((step.entropy.double().cpu() - entropy).abs() <= 4 * limit).all())
    assert torch.equal(step.ids.cpu().long(), ids.long())


def test_graphs_that_share_their_scratch():
    """Two captured steps, one scratch: replayed in turn, with new inputs and the same work eagerly in between, each gives
    what the eager step gives, every time."""
    scratch = _scratch()
    steps = [Step(scratch, seed) for seed in (3, 4)]
    graphs = []
    for step in steps:
        step.fill(5)
        step.run()                                          # (the library's own first calls)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step.run()
        graphs.append(graph)
    for turn in range(4):
        for step, graph in zip(steps, graphs):
            step.fill(10 + turn)
            step.clear()
            scratch.fill_(math.nan)
            graph.replay()
            replayed = [x.clone() for x in step.results()]
            step.clear()
            step.run()
            torch.cuda.synchronize()
            for one, other in zip(replayed, step.results()):
                assert torch.equal(one, other)
    for step, graph in zip(steps, graphs):
        step.fill(20)
    for graph in graphs * 2:                                # (without waiting in between)
        graph.replay()
    for step in steps:
        replayed = [x.clone() for x in step.results()]
        step.run()
        for one, other in zip(replayed, step.results()):
            assert torch.equal(one, other)


def test_on_another_stream():
    """The step on a stream that is not the default one, behind work of that stream that makes its inputs."""
    step = Step(_scratch(), 6)
    step.fill(7)
    step.run()
    expected = [x.clone() for x in step.results()]
    step.clear()
    kept = step.qkv.clone()
    step.qkv.zero_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        slow = torch.zeros(1 << 26, device="cuda")
        for _ in range(20):
            slow.add_(1.0)
        step.qkv.copy_(kept)
        step.run()
        got = [x.clone() for x in step.results()]
    side.synchronize()
    for one, other in zip(got, expected):
        assert torch.equal(one, other)


def test_the_same_token_twice():
    """A token listed twice, a tile listed twice, a position stored twice with the same row: as once."""
    step = Step(_scratch(), 8)
    step.fill(9)
    step.run()
    expected = [x.clone() for x in step.results()]
    step.clear()
    twice = lambda x: torch.cat([x, x])
    step.scratch = torch.cat([step.scratch, step.scratch])
    step.singles, step.tile_item, step.tile_q0 = twice(step.singles), twice(step.tile_item), twice(step.tile_q0)
    step.run()
    for one, other in zip(step.results(), expected):
        assert torch.equal(one, other)


def test_pools_beyond_32_bits():
    """Pages that lie 4 GiB and more behind the pool's first: stored, read and attended like those of a small pool."""
    from pagedserve_amd.ops import kernels

    heads, dim, page, length = 2, 128, 64, 700
    row = kernels.int4_row_bytes(dim)
    pages = (9 << 29) // (heads * page * row)               # 4.5 GiB
    pools = [torch.empty((pages, heads, page, row), dtype=torch.uint8, device="cuda") for _ in range(2)]
    small = [torch.zeros((11, heads, page, row), dtype=torch.uint8, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(11)
    rows = [torch.randn(length, heads * dim, generator=g).to(BF16).cuda() for _ in range(2)]
    q = torch.randn(length, 4 * heads * dim, generator=g).to(BF16).cuda()
    ints = lambda values: torch.tensor(values, dtype=torch.int32).cuda()
    far, near = ints([[pages - 1 - 7 * i for i in range(11)]]), ints([[10 - i for i in range(11)]])
    index = ints([0] * length), ints(list(range(length)))
    outs = []
    for use, tables in ((pools, far), (small, near)):
        kernels.kv_write_int4(*rows, *use, *index, tables)
        back = [torch.zeros_like(x) for x in rows]
        kernels.kv_read_int4(*use, *back, *index, tables)
        single, portion = torch.zeros_like(q[:1]), torch.zeros_like(q[:64])
        kernels.attention_decode_int4(q[:1], *use, single, None, ints([length - 1]), tables, 4 * heads, 0.1, 2,
                                      torch.empty(4 * heads * 2 * (dim + 2)).cuda())
        kernels.attention_prefill_int4(q[:64], *use, portion, ints([0]), ints([0]), ints([0, 64]), ints([length]), tables,
                                       4 * heads, 0.1, max_kv_len=length)
        outs.append([*back, single, portion])
    for one, other in zip(*outs):
        assert torch.equal(one, other)
    expected = plain.held(rows[0].float().cpu()[-3:], heads)[2]
    assert torch.equal(outs[0][0][-3:].double().cpu(), expected)


def test_rows_of_logits_beyond_32_bits():
    """Rows 2^30 logits apart: the third begins 2^31 elements behind the first."""
    from pagedserve_amd.ops import kernels

    vocab, apart = 5000, 1 << 30
    rows = torch.as_strided(torch.empty(2 * apart + vocab, dtype=BF16, device="cuda"), (3, vocab), (apart, 1))
    dense = (torch.randn(3, vocab, generator=torch.Generator().manual_seed(12)) * 3).to(BF16).cuda()
    rows.copy_(dense)
    wanted = torch.tensor([0, 17, vocab - 1], dtype=torch.int32).cuda()
    results = []
    scratch = torch.empty(kernels.logprob_scratch(3, vocab, 4)).cuda()
    for logits in (rows, dense):
        out, best = torch.zeros(3).cuda(), torch.zeros(3, 4).cuda()
        ids = torch.zeros(3, 4, dtype=torch.int32).cuda()
        kernels.token_logprobs(logits, wanted, out, None, None, ids, best, scratch)
        results.append((out, best, ids))
    for one, other in zip(*results):
        assert torch.equal(one, other)

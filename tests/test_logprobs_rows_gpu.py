"""Log probabilities of rows that lie in memory in unusual ways."""

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 37, 5000, 70001])
def test_one_row_for_many_tokens(kind, vocab):
    """A row expanded to all tokens, and a single row whose stride says nothing."""
    from pagedserve_amd.ops import kernels

    rows = 40
    logits = (torch.randn(vocab, generator=torch.Generator().manual_seed(vocab)) * 3).to(kind)
    top = min(5, vocab)
    tokens = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(1)).int()
    expected = plain.logprobs(logits.expand(rows, vocab), tokens, top)
    on = logits.cuda()
    for given, count in ((on.expand(rows, vocab), rows), (on.view(vocab, 1).t(), 1)):
        out, entropy, ranks = torch.zeros(count).cuda(), torch.zeros(count).cuda(), torch.zeros(count, dtype=torch.int32).cuda()
        ids, best = torch.zeros(count, top, dtype=torch.int32).cuda(), torch.zeros(count, top).cuda()
        partial = torch.zeros(max(1, kernels.logprob_scratch(count, vocab, top))).cuda()
        kernels.token_logprobs(given, tokens[:count].cuda(), out, entropy, ranks, ids, best, partial)
        # sums of `vocab` floats: errors that add up as their square root, of numbers up to 16
        allowed = 2.0 ** -23 * (16 + vocab ** 0.5) * (1 + expected[0][:count].abs())
        assert bool(((out.double().cpu() - expected[0][:count]).abs() <= allowed).all())
        assert bool(((entropy.double().cpu() - expected[1][:count]).abs() <= 2 * allowed * (1 + expected[1][:count])).all())
        assert torch.equal(ranks.long().cpu(), expected[2][:count]) and torch.equal(ids.long().cpu(), expected[3][:count])
        assert bool(((best.double().cpu() - expected[4][:count]).abs()
                     <= 2.0 ** -23 * (16 + vocab ** 0.5) * (1 + expected[4][:count].abs())).all())

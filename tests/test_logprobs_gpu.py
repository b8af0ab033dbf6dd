"""Log probabilities of given tokens on the GPU against plain formulas in 64 bits."""

import math

import pytest
import torch

import plain_int4 as plain

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _run(logits, tokens, top, **wanted):
    from pagedserve_amd.ops import kernels

    rows, vocab = logits.shape
    out = torch.full((rows + 1,), 5.0).cuda()
    entropy = torch.full((rows + 1,), 5.0).cuda()
    ranks = torch.full((rows + 1,), 5, dtype=torch.int32).cuda()
    ids = torch.full((rows, top), -7, dtype=torch.int32).cuda() if top else None
    best = torch.full((rows, top), 5.0).cuda() if top else None
    partial = torch.full((kernels.logprob_scratch(rows, vocab, top),), math.nan).cuda()
    kernels.token_logprobs(logits, tokens.cuda(), out[:rows], entropy[:rows], ranks[:rows], ids, best, partial)
    assert out[rows] == 5.0 and entropy[rows] == 5.0 and ranks[rows] == 5
    return out[:rows].cpu(), entropy[:rows].cpu(), ranks[:rows].cpu(), ids.cpu() if top else None, best.cpu() if top else None


def _check(logits, tokens, top, found):
    """Whole numbers exactly; a log probability within a float's rounding of its three terms (the logit and the maximum, whose
    difference is exact or rounded once, and the logarithm of a sum of n terms, rounded once each and scaled up to 12 times
    on the way); the entropy the same, times the spread of the logits that its sum weighs."""
    log_p, entropy, rank, ids, best = plain.logprobs(logits, tokens, top)
    spread = (logits.double().cpu().nan_to_num(neginf=0.0).amax(-1) - log_p).abs().nan_to_num(posinf=0.0)
    sums = 2.0 ** -24 * (16 + logits.shape[1] ** 0.5)
    limit = 2.0 ** -23 * log_p.abs() + 2 * sums
    assert bool(((found[0].double() - log_p).abs() <= limit).all()), (found[0].double() - log_p).abs().max()
    # (of the terms (x - M) e^(x - M) none is larger than 1 / e beside a Z of at least 1)
    assert bool(((found[1].double() - entropy).abs() <= 4 * sums * (1 + entropy)).all())
    assert torch.equal(found[2].long(), rank)
    if top:
        assert torch.equal(found[3].long(), ids)
        limit = 2.0 ** -23 * best.abs() + 2 * sums
        assert bool(((found[4].double() - best).abs() <= limit).all())
    del spread


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 2), (3, 5, 5), (7, 31, 8), (1, 300, 20), (300, 513, 3), (5, 4097, 32), (2, 50257, 5), (33, 50257, 20),
    (260, 50257, 1), (1, 131073, 7), (3, 160000, 20), (300, 70001, 0), (4, 1000, 0)])
def test_log_probabilities(kind, rows, vocab, top):
    g = torch.Generator().manual_seed(rows * 1000 + vocab)
    logits = (torch.randn((rows, vocab), generator=g) * 3.0).to(kind)
    tokens = torch.randint(0, vocab, (rows,), generator=g).to(torch.int32)
    tokens[::2] = logits[::2].float().argmax(-1).int()
    wide = torch.zeros((rows, vocab + 3), dtype=kind)
    wide[:, 1:1 + vocab] = logits
    # contiguous rows, rows within a wider buffer (and off its alignment)
    for given in (logits.cuda(), wide.cuda()[:, 1:1 + vocab]):
        _check(logits, tokens, top, _run(given, tokens, top))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("vocab", [40, 3000, 50257, 140000])
def test_equal_logits(kind, vocab):
    """Rows of one value, of two values, of rising and falling steps: the lower id comes first, and counts as more likely."""
    top = 20
    row = torch.arange(vocab)
    logits = torch.stack((torch.full((vocab,), 2.0), (row % 2).float(), (row // 7 % 5).float(), -(row // 1000).float(),
                          (row // 1000).float(), torch.where(row % 3 == 0, 0.0, -0.0))).to(kind)
    tokens = torch.tensor([vocab - 1, 0, 5, vocab // 2, 3, 1], dtype=torch.int32)
    logits[5] = 0.0
    logits[5, ::3] = -0.0
    _check(logits, tokens, top, _run(logits.cuda(), tokens, top))


@pytest.mark.parametrize("vocab", [9, 700, 50257])
def test_masked_logits(vocab):
    """Logits of minus infinity and of the type's lowest value; rows with one token left; the given token among them."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn((6, vocab), generator=g)
    logits[0, ::2] = -math.inf
    logits[1, 1:] = -math.inf
    logits[2, :-1] = torch.finfo(F32).min
    logits[3, vocab // 2:] = torch.finfo(F32).min
    logits[4] = torch.finfo(F32).min
    logits[5] *= 1e30
    tokens = torch.tensor([1, 0, vocab - 1, 0, vocab - 1, 2], dtype=torch.int32)
    found = _run(logits.cuda(), tokens, min(4, vocab))
    log_p, entropy, rank, ids, best = plain.logprobs(logits, tokens, min(4, vocab))
    assert torch.equal(found[2].long(), rank) and torch.equal(found[3].long(), ids)
    tolerance = 2.0 ** -23 * log_p.abs() + 2.0 ** -23 * (16 + vocab ** 0.5)
    assert bool(((found[0].double() - log_p).abs() <= tolerance).all())
    assert bool(((found[1].double() - entropy).abs() <= 2.0 ** -22 * (16 + vocab ** 0.5) * (1 + entropy)).all())
    finite = best.abs() < 1e38
    assert bool(((found[4].double() - best).abs()[finite] <= 2.0 ** -22 * best.abs()[finite] + 2.0 ** -23 * (16 + vocab ** 0.5)).all())
    # a given token that cannot come
    tokens[0] = 0
    assert _run(logits.cuda(), tokens, 1)[0][0] == -math.inf


def test_rows_without_a_distribution_and_without_a_token():
    logits = torch.randn((7, 100), generator=torch.Generator().manual_seed(3))
    logits[0] = -math.inf
    logits[1, 50] = math.nan
    logits[2, 9] = math.inf
    tokens = torch.tensor([5, 5, 5, -1, 100, -2, 1 << 30], dtype=torch.int32)
    out, entropy, ranks, ids, best = _run(logits.cuda(), tokens, 3)
    assert out[:3].isnan().all() and entropy[:3].isnan().all() and best[:3].isnan().all()
    assert ids[0].tolist() == [0, 1, 2] and ids[2, 0] == 9 and 50 not in ids[1].tolist()
    assert out[3] == 0 and out[4:].isnan().all() and ranks[3:].tolist() == [-1] * 4
    _, expected, _, expected_ids, _ = plain.logprobs(logits[3:], torch.zeros(4, dtype=torch.int32), 3)
    torch.testing.assert_close(entropy[3:].double(), expected, rtol=1e-5, atol=1e-5)
    assert torch.equal(ids[3:].long(), expected_ids)


def test_only_what_is_wanted():
    from pagedserve_amd.ops import kernels

    logits = torch.randn((2, 1000), generator=torch.Generator().manual_seed(4)).cuda()
    tokens = torch.tensor([3, 999], dtype=torch.int32)
    out = torch.zeros(2).cuda()
    partial = torch.zeros(kernels.logprob_scratch(2, 1000, 0)).cuda()
    kernels.token_logprobs(logits, tokens.cuda(), out, partial=partial)
    torch.testing.assert_close(out.double().cpu(), plain.logprobs(logits, tokens, 1)[0], rtol=1e-6, atol=1e-6)
    kernels.token_logprobs(logits[:0], tokens.cuda()[:0], out[:0])

"""How texts are taken through the engine to be scored, and the cache manager's pools in 4 bits: without a GPU, over an
engine that only keeps account."""

from types import SimpleNamespace
from unittest import mock

import pytest
import torch

import main
import plain_int4
from pagedserve_amd.cache.manager import CacheGroupSpec, CacheManager
from pagedserve_amd.engine import scoring

VOCAB = 23


def _row(tokens):
    """The logits behind these tokens: a number of them all, of their order, and of nothing else."""
    g = torch.Generator().manual_seed(hash(tuple(tokens)) % (1 << 31))
    return torch.randn(VOCAB, generator=g) * 2


class _Engine:
    """The engine's account of requests and pages; logits from ``_row``."""

    def __init__(self, pages=12, page_size=8, max_requests=3, max_step_tokens=16, window=0, fail_at=None):
        self.cache = CacheManager([CacheGroupSpec((0,), 1, 32, window)], pages, page_size, max_requests, torch.float32, "cpu",
                                  max_positions=pages * page_size, allocate_pools=False)
        self.max_positions, self.max_requests, self.max_step_tokens = pages * page_size, max_requests, max_step_tokens
        self.spec = SimpleNamespace(vocab_size=VOCAB)
        self.device = torch.device("cpu")
        self.texts, self.steps, self.fail_at = {}, [], fail_at

    def is_live(self, request):
        return request in self.cache.requests

    def finish(self, request):
        self.cache.release(request)
        del self.texts[request]

    def step(self, entries):
        self.steps.append([(entry.request_id, len(entry.tokens), list(entry.want)) for entry in entries])
        assert sum(len(entry.tokens) for entry in entries) <= self.max_step_tokens
        rows = []
        for entry in entries:
            if not self.is_live(entry.request_id):
                self.cache.admit(entry.request_id)
                self.texts[entry.request_id] = []
            text = self.texts[entry.request_id]
            for place, token in enumerate(entry.tokens):
                text.append(token)
                if place in entry.want:
                    rows.append(_row(text))
            self.cache.grow(entry.request_id, len(text))
            self.cache.commit(entry.request_id, len(text))
        if self.fail_at is not None and len(self.steps) == self.fail_at:
            raise RuntimeError("a step failed")
        return SimpleNamespace(logits=torch.stack(rows) if rows else torch.empty(0, VOCAB))


@pytest.fixture(autouse=True)
def plain_kernels():
    def token_logprobs(logits, tokens, out, entropy, ranks, ids, best, partial):
        top = 0 if ids is None else ids.shape[1]
        log_p, spread, rank, top_ids, top_p = plain_int4.logprobs(logits, tokens, top)
        out.copy_(log_p)
        entropy.copy_(spread)
        ranks.copy_(rank)
        if top:
            ids.copy_(top_ids)
            best.copy_(top_p)

    with mock.patch.object(scoring.kernels, "token_logprobs", token_logprobs), \
            mock.patch.object(scoring.kernels, "logprob_scratch", lambda *sizes: 0):
        yield


def _expected(text, top):
    rows = [plain_int4.logprobs(_row(text[:i])[None], torch.tensor([text[i]]), top) for i in range(1, len(text))]
    return [[float(row[which][0]) for row in rows] for which in range(3)], [
        list(zip(row[3][0].tolist(), row[4][0].tolist())) for row in rows]


@pytest.mark.parametrize("top", [0, 4])
@pytest.mark.parametrize("lengths,options", [
    ((1,), {}), ((2,), {}), ((16,), {}), ((17,), {}), ((40, 3, 16, 1, 15, 2), {}), ((5,) * 9, {}), ((96,), {}),
    ((90, 90), {}), ((20, 70, 20), {"max_requests": 1}), ((30, 8, 8, 50), {"max_step_tokens": 5}), ((60, 3, 60), {"window": 9})])
def test_every_token_of_every_text_is_scored_once(lengths, options, top):
    engine = _Engine(**options)
    g = torch.Generator().manual_seed(sum(lengths))
    texts = [torch.randint(0, VOCAB, (n,), generator=g).tolist() for n in lengths]
    found = scoring.score_tokens(engine, texts, top)
    for text, scores in zip(texts, found):
        (logprobs, entropies, ranks), alternatives = _expected(text, top)
        assert scores.token_ids == text
        assert scores.logprobs[1:] == pytest.approx(logprobs, abs=1e-5)
        assert scores.entropies[1:] == pytest.approx(entropies, abs=1e-5)
        assert scores.ranks[1:] == ranks and scores.logprobs[0] is None
        assert scores.total == pytest.approx(sum(logprobs), abs=1e-4)
        if not top:
            assert scores.alternatives is None
            continue
        assert [[i for i, _ in row] for row in scores.alternatives[1:]] == [[i for i, _ in row] for row in alternatives]
        assert [p for row in scores.alternatives[1:] for _, p in row] == pytest.approx(
            [p for row in alternatives for _, p in row], abs=1e-5)
    assert not engine.cache.requests and not engine.texts
    engine.cache.check_invariants()


def test_short_texts_share_a_step():
    engine = _Engine()
    scoring.score_tokens(engine, [[1, 2, 3, 4, 5]] * 3)
    assert len(engine.steps) == 1


def test_live_requests_stay():
    """Slots and pages that others hold are not taken; what cannot be placed is an error that leaves nothing behind."""
    engine = _Engine(pages=6)
    engine.cache.admit("other")
    engine.texts["other"] = []
    engine.cache.grow("other", 20)
    engine.cache.commit("other", 20)
    scoring.score_tokens(engine, [[1] * 20, [2] * 24])
    assert list(engine.cache.requests) == ["other"] and engine.cache.length("other") == 20
    with pytest.raises(RuntimeError, match="no pages or slots"):
        scoring.score_tokens(engine, [[1, 2], [1] * 25])
    assert list(engine.cache.requests) == ["other"]


def test_a_failing_step_leaves_nothing():
    engine = _Engine(fail_at=2)
    with pytest.raises(RuntimeError, match="a step failed"):
        scoring.score_tokens(engine, [[1] * 40, [2] * 3])
    assert not engine.cache.requests


@pytest.mark.parametrize("texts,top,message", [([[]], 0, "needs a token"), ([[1] * 97], 0, "97 tokens"), ([[1]], 24, "alternatives"),
                                               ([[1]], -1, "alternatives")])
def test_what_is_refused(texts, top, message):
    with pytest.raises(ValueError, match=message):
        scoring.score_tokens(_Engine(), texts, top)


def test_pools_in_4_bits():
    groups = [CacheGroupSpec((0, 1), 3, 48), CacheGroupSpec((2,), 2, 64, window=9)]
    cache = CacheManager(groups, 5, 8, 2, torch.bfloat16, "cpu", cache_format="int4")
    assert [tuple(pool.shape) for pool in cache.key_pools] == [(2, 5, 3, 8, 36), (1, 5, 2, 8, 36)]
    assert all(pool.dtype == torch.uint8 for pool in cache.key_pools + cache.value_pools)
    assert cache.key_pools[0].data_ptr() != cache.value_pools[0].data_ptr()
    assert cache.bytes_per_page(0) == 2 * 3 * 8 * 72 and cache.bytes_per_page(1) == 2 * 8 * 72
    assert CacheManager(groups, 5, 8, 2, torch.bfloat16, "cpu").bytes_per_page(0) == 2 * 3 * 8 * 2 * 48 * 2
    for bad, page, message in ((dict(cache_format="int8"), 8, "known: model, int4"), (dict(cache_format="int4"), 12, "multiple of 8")):
        with pytest.raises(ValueError, match=message):
            CacheManager(groups, 5, page, 2, torch.bfloat16, "cpu", **bad)
    for group in (CacheGroupSpec((0,), 1, 32, values_in_keys=True), CacheGroupSpec((0,), 1, 32, value_dim=16)):
        with pytest.raises(ValueError, match="values of their own"):
            CacheManager([group], 5, 8, 2, torch.bfloat16, "cpu", cache_format="int4")


def test_command_line_options(capsys):
    args = main.parse_args(["--kv-cache-dtype", "int4", "--score", "--prompt-ids", "1 2"])
    assert args.kv_cache_dtype == "int4" and args.score == 0
    assert main.parse_args(["--score", "7", "--prompt", "x"]).score == 7 and main.parse_args([]).score is None
    for bad in (["--score", "33", "--prompt", "x"], ["--score"], ["--kv-cache-dtype", "int2"]):
        with pytest.raises(SystemExit):
            main.parse_args(bad)
    capsys.readouterr()


def test_layers_that_take_no_cache_in_4_bits_are_refused():
    """Those that norm, rotate or gate queries and keys in a launch of their own, and those whose values are something else."""
    from pagedserve_amd.parts.attention import Attention

    plain = Attention(64, torch.float32, 4, 2, 16, 0.25)
    assert plain.takes_int4_cache
    assert Attention(64, torch.float32, 4, 2, 16, 0.25, sink=True, window=9, score_cap=3.0).takes_int4_cache
    for option in (dict(rotary_dims=8), dict(qk_norm=True), dict(head_gate=True), dict(values_from_keys=True), dict(value_dim=8),
                   dict(logistic=True), dict(head_norm=True)):
        assert not Attention(64, torch.float32, 4, 2, 16, 0.25, **option).takes_int4_cache

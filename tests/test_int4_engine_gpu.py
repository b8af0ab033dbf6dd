"""The engine over a cache in 4 bits, and texts scored over it: the operators together, as they are used."""

import math
import os
import subprocess
import sys

import pytest
import torch

import helpers
import int4_models
import plain_gpt2
import plain_int4

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# Seeds whose keys and values keep 4e-5 of a step from the borders between codes (float products of this size are off by some 1e-6
# of their values, 8e-6 of a step).
REQUESTS = {"A": (910, (40, 21, 1)), "B": (901, (33, 60, 2))}


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    base = tmp_path_factory.mktemp("int4_models")
    return {which: helpers.tiny_folder(base, which) for which in ("A", "B")}


def _requests(which, config):
    seed, lengths = REQUESTS[which]
    return {i: helpers.random_tokens(n, config["vocab_size"], seed + i) for i, n in enumerate(lengths)}


def _engine(folder, page_size, dtype="float32", kv_cache_dtype="int4", **options):
    from pagedserve_amd.engine import Engine
    from pagedserve_amd.model import load_model

    model, _ = load_model(folder, dtype=getattr(torch, dtype), device="cuda")
    return Engine(model, num_pages=options.pop("num_pages", 40), page_size=page_size, max_requests=4, max_step_tokens=256,
                  kv_cache_dtype=kv_cache_dtype, **options)


@pytest.mark.parametrize("trace", ["whole", "portions", "mixed", "tail_decoded"])
@pytest.mark.parametrize("which", ["A", "B"])
def test_logits_in_32_bit(models, which, trace):
    """The plain model over what the cache holds, under every cut of the work (heads of 16 and of 48, pages of 8 and 16)."""
    folder, config, page_size = models[which]
    requests = _requests(which, config)
    raw, weights = plain_gpt2.read_model_folder(folder)
    margins = []
    with int4_models.cache_in_4_bits(margins):
        reference = {rid: plain_gpt2.forward_logits(raw, weights, tokens) for rid, tokens in requests.items()}
    assert min(margins) > 3e-5
    engine = _engine(folder, page_size)
    assert engine.cache.key_pools[0].dtype == torch.uint8
    steps = getattr(helpers, f"trace_{trace}")(requests)
    rows = helpers.replay_in_process(engine, steps)
    worst, scale, where = helpers.max_error(rows, reference)
    assert worst <= 2e-5 * scale, (worst, scale, where)
    # and it is not what the cache of the model's type gives
    with_model = {rid: plain_gpt2.forward_logits(raw, weights, tokens) for rid, tokens in requests.items()}
    assert helpers.max_error(rows, with_model)[0] > 1e-3 * scale


@pytest.mark.parametrize("which", ["A", "B"])
def test_bfloat16_runs_under_every_cut(models, which):
    """Roundings of the model's activations turn codes here and there; what stays is that the logits follow the plain
    model's over such a cache about as closely as over its own, and that graphs change nothing but rounding."""
    folder, config, page_size = models[which]
    requests = _requests(which, config)
    raw, weights = plain_gpt2.read_model_folder(folder)
    with int4_models.cache_in_4_bits():
        reference = {rid: plain_gpt2.forward_logits(raw, weights, tokens) for rid, tokens in requests.items()}
    errors = []
    for graphs in (True, False):
        engine = _engine(folder, page_size, "bfloat16", use_graphs=graphs)
        for trace in (helpers.trace_mixed, helpers.trace_tail_decoded, helpers.trace_portions):
            rows = helpers.replay_in_process(engine, trace(requests))
            difference = torch.stack([row - reference[rid][at] for (rid, at), row in rows.items()])
            expected = torch.stack([reference[rid][at] for rid, at in rows])
            errors.append(float(difference.norm() / expected.norm()))
        assert not engine.cache.requests
    assert max(errors) < 0.15, errors


@pytest.mark.parametrize("dtype,limit", [("bfloat16", 0.15), ("float32", 2e-3)])
def test_long_contexts(tmp_path, dtype, limit):
    """Portions and single tokens behind hundreds of keys, where both are cut into ranges, with and without graphs.  (In
    32-bit a code that turns moves a logit by some thousandth; tests with margins hold the rest to rounding.)"""
    config = dict(helpers.TINY_A, n_positions=1024)
    folder = helpers.write_folder(os.path.join(str(tmp_path), "long"), config, helpers.lively_tensors(config, 5))
    requests = {i: helpers.random_tokens(n, config["vocab_size"], 950 + i) for i, n in enumerate((900, 640, 3))}
    raw, weights = plain_gpt2.read_model_folder(folder)
    with int4_models.cache_in_4_bits():
        reference = {rid: plain_gpt2.forward_logits(raw, weights, tokens) for rid, tokens in requests.items()}
    for graphs in (True, False):
        engine = _engine(folder, 16, dtype, use_graphs=graphs, num_pages=120)
        rows = helpers.replay_in_process(engine, helpers.trace_mixed(requests, portion=(60, 33, 129, 2), decode_tail=24))
        difference = torch.stack([row - reference[rid][at] for (rid, at), row in rows.items()])
        expected = torch.stack([reference[rid][at] for rid, at in rows])
        assert float(difference.norm() / expected.norm()) < limit
        assert len(rows) == 1543 and not engine.cache.requests


def test_generated_tokens_are_the_plain_models(models):
    """Greedy decoding through the scheduler, its graphs and the entry point, in 32-bit."""
    from pagedserve_amd.engine.llm import LLM
    from pagedserve_amd.sampling import SamplingParams

    folder, config, page_size = models["A"]
    prompts = [helpers.random_tokens(n, config["vocab_size"], 300 + i) for i, n in enumerate((5, 17, 31))]
    raw, weights = plain_gpt2.read_model_folder(folder)
    with int4_models.cache_in_4_bits():
        expected = [plain_gpt2.greedy_generate(raw, weights, prompt, 12) for prompt in prompts]
    for graphs in (True, False):
        llm = LLM(folder, dtype="float32", block_size=page_size, num_kv_pages=40, max_batch_size=4, eos_token_id=None,
                  kv_cache_dtype="int4", enable_hip_graphs=graphs)
        outputs = llm.generate(prompts, SamplingParams(max_new_tokens=12))
        assert [output.token_ids for output in outputs] == expected
        assert bool(llm.engine.graphs_captured) == graphs
        llm.engine.cache.check_invariants()


@pytest.mark.parametrize("kv_cache_dtype", ["model", "int4"])
def test_scores(models, kv_cache_dtype):
    """Log probabilities, entropies, ranks and alternatives of given texts against the plain model's, over either cache; what
    they say of the cache in 4 bits is what it costs."""
    from pagedserve_amd.engine.llm import LLM

    folder, config, page_size = models["A"]
    texts = list(_requests("A", config).values()) + [helpers.random_tokens(100, config["vocab_size"], 77)]
    raw, weights = plain_gpt2.read_model_folder(folder)
    llm = LLM(folder, dtype="float32", block_size=page_size, num_kv_pages=20, max_batch_size=2, eos_token_id=None,
              kv_cache_dtype=kv_cache_dtype, max_num_batched_tokens=64)
    # (the text that went in last has no margin: it is compared over the model's cache only)
    found = llm.score(texts if kv_cache_dtype == "model" else texts[:3], top=5)
    for text, scores in zip(texts, found):
        if kv_cache_dtype == "int4":
            with int4_models.cache_in_4_bits():
                logits = plain_gpt2.forward_logits(raw, weights, text)
        else:
            logits = plain_gpt2.forward_logits(raw, weights, text)
        assert scores.token_ids == text
        assert scores.logprobs[0] is scores.ranks[0] is scores.entropies[0] is scores.alternatives[0] is None
        assert len(scores.logprobs) == len(scores.ranks) == len(scores.entropies) == len(scores.alternatives) == len(text)
        if len(text) == 1:
            assert scores.total == 0
            continue
        # float logits, off by 2e-5 of the largest: a log probability and an entropy move by twice that
        allowed = 4e-5 * float(logits.abs().max())
        log_p, entropy, rank, ids, best = plain_int4.logprobs(logits[:-1], torch.tensor(text[1:], dtype=torch.int32), 5)
        assert (torch.tensor(scores.logprobs[1:]).double() - log_p).abs().max() <= allowed
        assert (torch.tensor(scores.entropies[1:]).double() - entropy).abs().max() <= 8 * allowed
        assert abs(scores.total - float(log_p.sum())) <= allowed * len(text)
        got = torch.tensor([[p for _, p in row] for row in scores.alternatives[1:]]).double()
        assert (got - best).abs().max() <= allowed
        # (ranks and alternatives turn only where two logits are closer than that)
        gaps = (logits[:-1].sort(dim=-1).values.diff(dim=-1).amin(-1)) > 4 * allowed
        assert [r for r, clear in zip(scores.ranks[1:], gaps) if clear] == [int(r) for r, clear in zip(rank, gaps) if clear]
        same = [[i for i, _ in row] == expected.tolist() for row, expected in zip(scores.alternatives[1:], ids)]
        assert sum(same) >= 0.9 * len(same)
    assert not llm.engine.cache.requests
    llm.engine.cache.check_invariants()


def test_scores_of_bfloat16_over_both_caches(models):
    """A text scored over the model's cache and over the one in 4 bits, with and without a bad token in it."""
    from pagedserve_amd.engine.llm import LLM

    folder, config, page_size = models["B"]
    text = helpers.random_tokens(200, config["vocab_size"], 5)
    totals = {}
    for kv_cache_dtype in ("model", "int4"):
        llm = LLM(folder, dtype="bfloat16", block_size=page_size, num_kv_pages=40, max_batch_size=2, eos_token_id=None,
                  kv_cache_dtype=kv_cache_dtype)
        once, again = llm.score([text])[0], llm.score([text], top=3)[0]
        assert once.alternatives is None and all(math.isfinite(p) for p in once.logprobs[1:])
        assert abs(once.total - again.total) <= 1e-2 * abs(once.total)
        totals[kv_cache_dtype] = once.total
    assert totals["model"] != totals["int4"]
    assert abs(totals["model"] - totals["int4"]) < 0.1 * abs(totals["model"])


def test_a_page_of_an_ended_request_is_used_again(models):
    """Pages come with what another request left in them; nothing of it is read."""
    folder, config, page_size = models["A"]
    engine = _engine(folder, page_size, "bfloat16", num_pages=8)
    text = helpers.random_tokens(60, config["vocab_size"], 9)
    first = helpers.replay_in_process(engine, helpers.trace_whole({"x": text}))
    for pool in engine.cache.key_pools + engine.cache.value_pools:
        pool.fill_(0xff)                       # NaN steps everywhere
    again = helpers.replay_in_process(engine, helpers.trace_whole({"y": text}))
    for (_, at), row in first.items():
        assert bool(torch.isfinite(again[("y", at)]).all())
        torch.testing.assert_close(again[("y", at)], row, rtol=1e-3, atol=1e-3)


def test_what_is_refused(models, tmp_path):
    import kosesun_models
    from pagedserve_amd.engine.llm import LLM

    folder, config, page_size = models["A"]
    with pytest.raises(ValueError, match="multiple of 8"):
        LLM(folder, block_size=12, num_kv_pages=8, kv_cache_dtype="int4")
    other, _, _, page = kosesun_models.folder_of(str(tmp_path), "A")
    with pytest.raises(ValueError, match="does not take a cache in 4 bits"):
        LLM(other, block_size=page, num_kv_pages=8, kv_cache_dtype="int4")
    llm = LLM(folder, block_size=page_size, num_kv_pages=4, max_batch_size=2, kv_cache_dtype="int4")
    for texts, top, message in (([[]], 0, "needs a token"), ([[1] * 200], 0, "tokens"), ([[1, 2]], 33, "alternatives"),
                                ([[1, 2]], -1, "alternatives")):
        with pytest.raises(ValueError, match=message):
            llm.score(texts, top)
    with pytest.raises(ValueError, match="outside"):
        llm.score([[1, config["vocab_size"]]])
    assert not llm.engine.cache.requests


def test_the_cache_is_sized_by_its_form(models):
    """The same memory holds 3.5 times the pages (heads of 16 take the 18 bytes of 32 dimensions, where bfloat16 takes 32)."""
    from pagedserve_amd.engine.llm import LLM

    folder, _, page_size = models["A"]
    pages = {}
    for kv_cache_dtype in ("model", "int4"):
        llm = LLM(folder, dtype="bfloat16", block_size=page_size, kv_cache_memory_mb=1, max_batch_size=2,
                  kv_cache_dtype=kv_cache_dtype)
        pages[kv_cache_dtype] = llm.engine.cache.pools[0].num_pages
        assert llm.engine.cache.bytes_per_page(0) == (2 * 2 * 4 * page_size * (32 if kv_cache_dtype == "model" else 18))
    assert pages["int4"] == 2 ** 20 // (16 * page_size * 18) and pages["model"] == 2 ** 20 // (16 * page_size * 32)


def test_command_line_scores(models):
    folder, config, page_size = models["A"]
    command = [sys.executable, os.path.join(ROOT, "main.py"), "--model", folder, "--dtype", "bfloat16", "--num-kv-pages", "20",
               "--block-size", str(page_size), "--kv-cache-dtype", "int4", "--score", "2", "--prompt-ids", "5 17 3 99"]
    result = subprocess.run(command, capture_output=True, text=True, timeout=100)
    assert result.returncode == 0, result.stderr[-2000:]
    lines = result.stdout.strip().splitlines()
    assert lines[0].startswith("text 0: 4 tokens, log probability -")
    assert len(lines) == 5 and "rank" in lines[2] and "entropy" in lines[4]

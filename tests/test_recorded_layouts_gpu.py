"""Recorded steps with prompt portions: what a replay gives is bit for bit what the same launches give when they are made
directly, over the cache of the model's type and over the one in 4 bits."""

import os

import pytest
import torch

import helpers

pytestmark = pytest.mark.gpu

CONFIG = dict(helpers.TINY_A, n_positions=1024)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return helpers.write_folder(os.path.join(str(tmp_path_factory.mktemp("layouts")), "model"), CONFIG,
                                helpers.lively_tensors(CONFIG, 7))


def _engine(folder, dtype, cache, record_after):
    from pagedserve_amd.engine import Engine
    from pagedserve_amd.model import load_model

    model, _ = load_model(folder, dtype=getattr(torch, dtype), device="cuda")
    engine = Engine(model, num_pages=160, page_size=16, max_requests=4, max_step_tokens=640, kv_cache_dtype=cache)
    engine.record_after = record_after
    # (the largest step first: buffers are not replaced later)
    _step(engine, [("first", helpers.random_tokens(640, CONFIG["vocab_size"], 1))])
    engine.finish("first")
    return engine


def _step(engine, parts):
    """Logits at every place of every part ``(request, tokens)``."""
    from pagedserve_amd.engine import StepEntry

    logits = engine.step([StepEntry(rid, tokens, list(range(len(tokens)))) for rid, tokens in parts]).logits.clone()
    torch.cuda.synchronize()
    return logits


@pytest.mark.parametrize("cache", ["model", "int4"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_layouts_with_equal_sums_of_tiles(folder, dtype, cache):
    """As many tokens, requests and tiles in all, but other numbers of every size: each replays its own launches."""
    pairs = [((33, 33, 33), (2, 2, 95)), ((131, 97, 72), (137, 132, 31))]
    layouts = [counts for pair in pairs for counts in pair]
    texts = {counts: [helpers.random_tokens(count, CONFIG["vocab_size"], 31 * count + place)
                      for place, count in enumerate(counts)] for counts in layouts}
    rows = {}
    for record_after in (1 << 30, 1):
        engine = _engine(folder, dtype, cache, record_after)
        for turn in range(4):
            for counts in layouts:
                logits = _step(engine, list(enumerate(texts[counts])))
                for request in range(len(counts)):
                    engine.finish(request)
                if record_after > 1 and turn == 0:
                    rows[counts] = logits
                else:
                    assert torch.equal(logits, rows[counts]), (counts, turn, record_after)
        summary = engine.graph_summary()
        assert not summary["capture_failures"]
        assert summary["captures"] == summary["captured_graphs"] == (4 if record_after == 1 else 0), summary
        assert summary["graph_replays"] == (12 if record_after == 1 else 0), summary


@pytest.mark.parametrize("cache", ["model", "int4"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_portions_beside_single_tokens_behind_hundreds_of_keys(folder, dtype, cache):
    """Steps with a portion and single tokens, and with portions alone, whose keys are cut into ranges: recorded, replayed
    with other contexts under the same bound, and alternating, so that they pass the same scratch between them."""
    from pagedserve_amd.ops import kernels

    tokens = {rid: helpers.random_tokens(count, CONFIG["vocab_size"], 70 + rid) for rid, count in enumerate((1000, 900, 700))}
    if cache == "int4" and dtype == "bfloat16":
        heads = CONFIG["n_head"]
        assert kernels.prefill_int4_ranges(1, heads, 1024) > 1
        assert kernels.int4_decode_splits(torch.bfloat16, 2, heads, heads, CONFIG["n_embd"] // heads, 1024) > 1
    steps = [[(0, 600)], [(1, 520)], [(2, 530)]]
    for _ in range(6):
        steps += [[(0, 40), (1, 1), (2, 1)], [(1, 25), (2, 9)]]
    rows = {}
    for record_after in (1 << 30, 2):
        engine = _engine(folder, dtype, cache, record_after)
        at = {rid: 0 for rid in tokens}
        for number, step in enumerate(steps):
            parts = []
            for rid, count in step:
                parts.append((rid, tokens[rid][at[rid]:at[rid] + count]))
                at[rid] += count
            logits = _step(engine, parts)
            if record_after > 2:
                rows[number] = logits
            else:
                assert torch.equal(logits, rows[number]), number
        if record_after == 2:
            keys = list(engine._graphs)
            assert not engine.graph_summary()["capture_failures"]
            assert sorted((key[0], key[3]) for key in keys) == [(34, 0), (42, 2)], keys
            assert engine.graph_summary()["graph_replays"] == 8

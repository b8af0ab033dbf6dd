"""The engine over a cache in 4 bits with heads of many sizes: every kernel that such a size goes to, as a model calls it."""

import os

import pytest
import torch

import helpers
import int4_models
import plain_gpt2

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,dim,page", [(4, 7, 8), (3, 20, 8), (2, 40, 16), (2, 80, 16), (4, 128, 16), (2, 160, 24),
                                            (2, 256, 64), (1, 250, 8), (16, 96, 16)])
def test_portions_and_single_tokens(tmp_path, heads, dim, page):
    """Portions beside single tokens behind up to 300 keys, recorded at a layout's fourth step, against the plain model.  (The
    bounds are those of the engine's other tests: roundings turn codes, which is a whole step.)"""
    from pagedserve_amd.engine import Engine
    from pagedserve_amd.model import load_model

    config = dict(helpers.TINY_A, n_positions=512, n_embd=heads * dim, n_head=heads, n_inner=64)
    folder = helpers.write_folder(os.path.join(str(tmp_path), "model"), config, helpers.lively_tensors(config, 5))
    requests = {i: helpers.random_tokens(n, config["vocab_size"], 50 + i) for i, n in enumerate((300, 170, 3))}
    raw, weights = plain_gpt2.read_model_folder(folder)
    with int4_models.cache_in_4_bits():
        reference = {rid: plain_gpt2.forward_logits(raw, weights, tokens) for rid, tokens in requests.items()}
    for dtype, limit in (("bfloat16", 0.15), ("float32", 2e-3)):
        model, _ = load_model(folder, dtype=getattr(torch, dtype), device="cuda")
        engine = Engine(model, num_pages=-(-700 // page) + 4, page_size=page, max_requests=4, max_step_tokens=256,
                        kv_cache_dtype="int4")
        engine.record_after = 3
        rows = helpers.replay_in_process(engine, helpers.trace_mixed(requests, portion=(60, 33, 90, 2), decode_tail=24))
        difference = torch.stack([row - reference[rid][at] for (rid, at), row in rows.items()])
        expected = torch.stack([reference[rid][at] for rid, at in rows])
        assert float(difference.norm() / expected.norm()) < limit, dtype
        assert not engine.graph_summary()["capture_failures"] and not engine.cache.requests

"""Which steps the engine takes for the same recorded launches, on the CPU: an engine whose forward pass and index copies are
stand-ins, so that only its account of layouts and recorded graphs runs."""

from types import SimpleNamespace
from unittest import mock

import pytest
import torch

from pagedserve_amd.cache.manager import CacheGroupSpec, CacheManager
from pagedserve_amd.engine import engine as engine_module
from pagedserve_amd.engine.engine import Engine, StepEntry
from pagedserve_amd.ops import kernels

TILES = (32, 64, 128)


class _Words:
    def __init__(self, words, memory=None, at=0):
        self.tensor = torch.zeros(words, dtype=torch.int32)

    def to_device(self, device, words):
        device[:words] = self.tensor[:words]


class _Event:
    def record(self, stream=None):
        pass

    def synchronize(self):
        pass

    def query(self):
        return True


class _Graph:
    """A recorded step."""

    begin = abort = staticmethod(lambda: None)

    def __init__(self):
        self.replays = self.nodes = 0

    def end(self):
        pass

    def launch(self):
        self.replays += 1

    def destroy(self):
        pass


@pytest.fixture
def engine():
    model = SimpleNamespace(spec=SimpleNamespace(max_positions=2048, vocab_size=50), device=torch.device("cpu"),
                            dtype=torch.float32, graph_safe=True, query_tiles=TILES, check_cache_format=lambda form: None,
                            cache_requirements=lambda: ([CacheGroupSpec((0,), 1, 32)], ()), cache_views=lambda cache: [])
    with mock.patch.object(torch.cuda, "is_available", lambda: True), \
            mock.patch.object(torch.cuda, "Event", _Event), \
            mock.patch.object(torch.cuda, "Stream", lambda device=None: None), \
            mock.patch.object(kernels, "HostWords", _Words), \
            mock.patch.object(kernels, "StepGraph", _Graph), \
            mock.patch.object(kernels, "TopChoice", lambda rows, device: None), \
            mock.patch.object(engine_module, "CacheManager", lambda *args, **options: CacheManager(
                *args, **options, allocate_pools=False)):
        made = Engine(model, num_pages=256, page_size=16, max_requests=8, max_step_tokens=512)
        made.launched = []

        def forward(ctx, rows, logits, wanted, greedy):
            made.launched.append(ctx.tokens)
            return logits[:wanted], None

        made._forward = forward
        yield made


def _run(engine, counts):
    """One step of new requests that bring so many tokens each; whether it was a replay."""
    entries = []
    for index, count in enumerate(counts):
        engine.cache.admit(index)
        engine.cache.grow(index, count)
        entries.append(StepEntry(index, [1] * count, [count - 1]))
    before = len(engine.launched)
    engine._run_step(entries)
    for index in range(len(counts)):
        engine.cache.release(index)
    return len(engine.launched) == before


@pytest.mark.parametrize("first,second", [((33, 33, 33), (2, 2, 95)), ((131, 97, 72), (137, 132, 31))])
def test_layouts_of_equal_sums_are_recorded_apart(engine, first, second):
    """As many tokens, requests and tiles in all, but not of every size: the arrays of the one lie where the other has
    something else, and its launches are of other sizes."""
    tiles = [tuple(sum(-(-count // size) for count in counts) for size in TILES) for counts in (first, second)]
    assert sum(first) == sum(second) and sum(tiles[0]) == sum(tiles[1]) and tiles[0] != tiles[1]
    engine.record_after = 2
    assert [_run(engine, first) for _ in range(4)] == [False, False, False, True]
    assert [_run(engine, second) for _ in range(4)] == [False, False, False, True]
    assert engine.graphs_captured == 2 and len(engine._graphs) == 2


def test_a_layout_that_comes_back_is_replayed(engine):
    """Portions of other lengths with the same tiles of every size share a recorded step."""
    engine.record_after = 1
    assert [_run(engine, counts) for counts in ((50, 60), (60, 50), (55, 55), (33, 77))] == [False, False, True, False]
    assert engine.graphs_captured == 1


def test_decoded_tokens_are_replayed_by_the_short_way(engine):
    """A token per request with its logits: recorded at its second step, replayed from then on without listing anything."""
    for index in range(3):
        engine.cache.admit(index)
        engine.cache.grow(index, 20)
        engine.cache.commit(index, 5 + index)
    packed = []
    pack = engine._pack
    engine._pack = lambda *args: packed.append(1) or pack(*args)
    for step in range(4):
        engine._run_step([StepEntry(index, [1], [0]) for index in range(3)])
    assert len(engine.launched) == 2 and engine.graphs_captured == 1 and len(packed) == 2

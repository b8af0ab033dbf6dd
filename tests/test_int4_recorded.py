"""Scratch of a recorded call over a cache in 4 bits, without a GPU."""

from types import SimpleNamespace
from unittest import mock

import pytest
import torch

from pagedserve_amd.ops import kernels
from test_int4 import _prompt, on_gpu  # noqa: F401


class _Entry:
    """A C entry that succeeds."""

    def __call__(self, *args):
        return 0


def test_no_scratch_of_the_call_in_a_recorded_one(on_gpu):  # noqa: F811
    """What a call allocates for itself is given back at its end; the replays of a recorded one would write there."""
    lib = SimpleNamespace(ps_graph_begin=_Entry(), ps_graph_end=_Entry(), ps_graph_abort=_Entry())
    ranges = dict(ranges=2)
    with mock.patch.object(kernels, "load_library", lambda: lib):
        kernels.attention_prefill_int4(**_prompt(**ranges))
        graph = kernels.StepGraph()
        for leave in (graph.end, kernels.StepGraph.abort):
            kernels.StepGraph.begin()
            with pytest.raises(kernels.KernelError, match="give it as partial"):
                kernels.attention_prefill_int4(**_prompt(**ranges))
            kernels.attention_prefill_int4(**_prompt(ranges=1))
            kernels.attention_prefill_int4(**_prompt(partial=torch.zeros(9), **ranges))
            leave()
        kernels.attention_prefill_int4(**_prompt(**ranges))
    assert len(on_gpu) == 6

"""Texts scored by an engine whose device is not the current one, without a GPU: kernels are launched on the current
device's stream, and refuse tensors of another."""

from contextlib import contextmanager
from unittest import mock

import torch

from pagedserve_amd.engine import scoring
from pagedserve_amd.ops import kernels


def test_the_engines_device_is_the_current_one_while_rows_are_scored():
    current, launched = [0], []

    @contextmanager
    def device_of(tensor):
        before, current[0] = current[0], tensor.device
        yield
        current[0] = before

    def token_logprobs(logits, *rest):
        launched.append((logits.device, current[0]))

    rows = scoring._Rows(4, 2, torch.device("cpu"))
    with mock.patch.object(torch.cuda, "device_of", device_of), \
            mock.patch.object(kernels, "token_logprobs", token_logprobs), \
            mock.patch.object(kernels, "logprob_scratch", lambda rows, vocab, top: 0):
        rows.score(torch.zeros(3, 20), [1, 2, 3])
    assert launched == [(torch.device("cpu"),) * 2] and current == [0]

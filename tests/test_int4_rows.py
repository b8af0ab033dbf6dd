"""Rows of unusual strides at the faces of the operators of a cache in 4 bits and of the log probabilities, without a GPU."""

from unittest import mock

import pytest
import torch

from pagedserve_amd.ops import kernels
from test_int4 import BF16, _c, _decode, _float_prompt, _ints, _logprobs, _prompt, _write, on_gpu  # noqa: F401


def _calls(function, args):
    found = []
    with mock.patch.object(kernels, "_call", lambda name, *given: found.append(given)):
        function(**args)
    return found[0]


def test_a_single_row_is_as_long_as_its_stride(on_gpu):  # noqa: F811
    """The stride of a single row means nothing: a column that was turned has 1."""
    def turned(n, kind=torch.float32):
        row = torch.zeros(n, dtype=kind).view(n, 1).t()
        assert row.shape == (1, n) and row.stride() == (1, 1)
        return row

    given = _calls(kernels.kv_write_int4, _write(k=turned(128), v=turned(128), tok_item=_ints(1), tok_pos=_ints(1)))
    assert given[2:4] == (128, 128)
    given = _calls(kernels.attention_decode_int4, _decode(q=turned(256, BF16), out=turned(256, BF16), tok_item=_ints(1), tok_pos=_ints(1)))
    assert given[1] == given[9] == 256
    given = _calls(kernels.token_logprobs, _logprobs(logits=turned(50), tokens=_ints(1), out=torch.zeros(1)))
    assert given[1:4] == (50, 1, 50)


@pytest.mark.parametrize("function,args,kind", [(kernels.attention_decode_int4, _decode, BF16),
                                                (kernels.attention_prefill_int4, _prompt, BF16),
                                                (kernels.attention_tiled_f32_int4, _float_prompt, torch.float32)])
def test_results_that_overlap_are_refused(on_gpu, function, args, kind):  # noqa: F811
    """Queries may share a row, results may not."""
    row = torch.zeros(256, dtype=kind)
    function(**args(q=row.expand(3, 256)))
    assert len(on_gpu) == 1
    for out in (row.expand(3, 256), torch.zeros(600, dtype=kind).as_strided((3, 256), (8, 1))):
        with pytest.raises(kernels.KernelError, match="overlap"):
            function(**args(out=out))
    assert len(on_gpu) == 1


def test_a_row_of_logits_for_many_tokens(on_gpu):  # noqa: F811
    """One distribution, several tokens asked about: the library takes rows that are all the same one."""
    given = _calls(kernels.token_logprobs, _logprobs(logits=torch.zeros(50).expand(3, 50)))
    assert given[1:4] == (0, 3, 50)
    # (scratch, which is missing, is asked for after the sizes)
    for ld, vocab, message in ((0, 200000, "too few"), (200000, 200000, "too few"), (199999, 200000, "bad sizes"), (-50, 50, "bad sizes")):
        status, error = _c("ps_token_logprobs", 0, ld, 3, vocab, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
        assert status == 1 and message in error

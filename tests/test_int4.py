"""What the operators of the cache in 4 bits and the log probabilities refuse, without a GPU: the checks of the Python
faces (on CPU tensors that claim to be on the device) and those at the C entries, which return before any launch."""

import ctypes
import os
from unittest import mock

import pytest
import torch

import kernel_code
import plain_int4 as plain
from pagedserve_amd.ops import kernels, library

BF16, F32 = torch.bfloat16, torch.float32


# (twice: where the current device is unknown, and where the tensors' is the current one)
@pytest.fixture(params=[None, -1])
def on_gpu(request):
    """CPU tensors pass the question where they live; whatever gets past the checks is caught."""
    launched = []
    with mock.patch.object(torch.Tensor, "is_cuda", property(lambda tensor: True)), \
            mock.patch.object(kernels, "_call", lambda name, *args: launched.append(name)), \
            mock.patch.object(kernels, "_stream", lambda: 0), \
            mock.patch.object(torch._C, "_cuda_getDevice", lambda: request.param, create=True), \
            mock.patch.object(kernels, "_check_prefill_constants", lambda: None):
        yield launched


def _ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _pools(kv_heads=2, dim=64, page=16, pages=4):
    return [torch.zeros(pages, kv_heads, page, kernels.int4_row_bytes(dim), dtype=torch.uint8) for _ in range(2)]


def _write(**changed):
    k_pool, v_pool = _pools()
    args = dict(k=torch.zeros(3, 128), v=torch.zeros(3, 128), k_pool=k_pool, v_pool=v_pool, tok_item=_ints(3),
                tok_pos=_ints(3), tables=_ints(1, 5))
    args.update(changed)
    return args


def _decode(**changed):
    k_pool, v_pool = _pools()
    args = dict(q=torch.zeros(3, 256, dtype=BF16), k_pool=k_pool, v_pool=v_pool, out=torch.zeros(3, 256, dtype=BF16),
                tok_item=_ints(3), tok_pos=_ints(3), tables=_ints(1, 5), heads=4, scale=0.125, splits=1)
    args.update(changed)
    return args


def _prompt(**changed):
    args = _decode(tile_item=_ints(1), tile_q0=_ints(1), cu_tokens=_ints(2), kv_lens=_ints(1))
    for name in ("tok_item", "tok_pos", "splits"):
        del args[name]
    args.update(changed)
    return args


def _float_prompt(**changed):
    args = _prompt(q=torch.zeros(3, 256), out=torch.zeros(3, 256))
    args.update(changed)
    return args


def _logprobs(**changed):
    args = dict(logits=torch.zeros(3, 50), tokens=_ints(3), out=torch.zeros(3))
    args.update(changed)
    return args


def test_what_they_take(on_gpu):
    kernels.kv_write_int4(**_write())
    kernels.kv_read_int4(**_write())
    kernels.attention_decode_int4(**_decode())
    kernels.attention_prefill_int4(**_prompt())
    kernels.token_logprobs(**_logprobs())
    kernels.attention_tiled_f32_int4(**_float_prompt())
    assert on_gpu == ["ps_kv_write_int4", "ps_kv_read_int4", "ps_attention_decode_int4", "ps_attention_prefill_int4",
                      "ps_token_logprobs", "ps_attention_tiled_f32_int4"]


@pytest.mark.parametrize("changed,message", [
    ({"v": torch.zeros(3, 128, dtype=BF16)}, "float32"), ({"k": torch.zeros(3, 64)}, "share a shape"),
    ({"k": torch.zeros(3, 126), "v": torch.zeros(3, 126)}, None), ({"k": torch.zeros(3, 130), "v": torch.zeros(3, 130)}, "do not fit"),
    ({"k_pool": torch.zeros(4, 2, 16, 36)}, "uint8"), ({"k_pool": _pools(pages=3)[0]}, "one shape"),
    ({"k_pool": _pools(page=12)[0], "v_pool": _pools(page=12)[0]}, "multiple of 8"),
    ({"k_pool": _pools(pages=0)[0], "v_pool": _pools(pages=0)[0]}, "empty"),
    ({"k_pool": torch.zeros(4 * 2 * 16 * 36 + 1, dtype=torch.uint8)[1:].view(4, 2, 16, 36)}, "16 bytes"),
    ({"tok_item": _ints(2)}, "item index"), ({"tok_pos": _ints(2)}, "position"), ({"tok_item": None}, "item index"),
    ({"tables": _ints(1, 5).long()}, "int32"), ({"tables": _ints(5, 2).t()}, "contiguous"),
    ({"k": torch.zeros(128, 3).t(), "v": torch.zeros(128, 3).t()}, "contiguous rows"),
    ({"k": torch.zeros(3, 128, dtype=torch.float16), "v": torch.zeros(3, 128, dtype=torch.float16)}, "not supported"),
    ({"k_pool": None}, "must be a tensor"), ({"v": [1.0]}, "must be a tensor"), ({"tok_pos": _ints(6)[::2]}, "contiguous")])
@pytest.mark.parametrize("function", [kernels.kv_write_int4, kernels.kv_read_int4])
def test_rows_refused(on_gpu, function, changed, message):
    if message is None:                                  # 63 dimensions take as many bytes as 64
        function(**_write(**changed))
        return
    with pytest.raises(kernels.KernelError, match=message):
        function(**_write(**changed))
    assert not on_gpu


def test_tensors_on_two_devices(on_gpu):
    """One tensor after the other claims another device than the first one's."""
    for function, args in ((kernels.kv_write_int4, _write()), (kernels.kv_read_int4, _write()),
                           (kernels.attention_decode_int4, _decode(tok_list=_ints(2), sink=torch.zeros(4), splits=2,
                                                                   partial=torch.zeros(4000))),
                           (kernels.attention_prefill_int4, _prompt(sink=torch.zeros(4), ranges=2, partial=torch.zeros(9))),
                           (kernels.attention_tiled_f32_int4, _float_prompt(sink=torch.zeros(4))),
                           (kernels.token_logprobs, _logprobs(entropy=torch.zeros(3), ranks=_ints(3), top_ids=_ints(3, 2),
                                                              top_logprobs=torch.zeros(3, 2), partial=torch.zeros(9)))):
        names = [name for name, value in args.items() if isinstance(value, torch.Tensor)]
        for name in names[1:]:
            other = args[name]
            with mock.patch.object(torch.Tensor, "get_device", lambda tensor: -2 if tensor is other else -1):
                with pytest.raises(kernels.KernelError, match="device"):
                    function(**args)
        assert not on_gpu
        function(**args)
        on_gpu.clear()


def test_tensors_that_are_not_on_the_current_device(on_gpu):
    with mock.patch.object(torch.Tensor, "get_device", lambda tensor: 1), \
            mock.patch.object(torch._C, "_cuda_getDevice", lambda: 0, create=True), \
            mock.patch.object(torch.cuda, "current_device", lambda: 0):
        with pytest.raises(kernels.KernelError, match="current device is 0"):
            kernels.kv_write_int4(**_write())


@pytest.mark.parametrize("changed,message", [
    ({"heads": 3}, "do not fit"), ({"heads": 0}, "do not fit"), ({"out": torch.zeros(3, 128, dtype=BF16)}, "rows must hold"),
    ({"out": torch.zeros(3, 256)}, "bfloat16"), ({"splits": 2}, "partial must be a tensor"),
    ({"splits": 2, "partial": torch.zeros(9, dtype=BF16)}, "partial"), ({"splits": 2, "partial": torch.zeros(9, 2)[:, 0]}, "contiguous"),
    ({"tok_item": None}, "row per token"), ({"tok_list": _ints(3).long()}, "int32"), ({"tok_list": _ints(6)[::2]}, "contiguous"),
    ({"sink": torch.zeros(3)}, "one float per head"), ({"softcap": -1.0}, "score cap"), ({"softcap": float("inf")}, "score cap"),
    ({"k_pool": _pools(dim=128)[0], "v_pool": _pools(dim=128)[0]}, "do not fit"),
    ({"store": (torch.zeros(3, 128), torch.zeros(3, 128))}, "bfloat16"), ({"store": (torch.zeros(2, 128, dtype=BF16),) * 2}, "stored are"),
    ({"store": (torch.zeros(3, 64, dtype=BF16),) * 2}, "stored are"), ({"store": (torch.zeros(3, 128, dtype=BF16),) * 2, "scale": -1.0, "tok_item": None}, "row per token"),
    ({"store": (torch.zeros(3, 128, dtype=BF16),) * 2}, "stored are"),
    ({"store": (torch.zeros(3, 128, dtype=BF16),) * 2, "tok_item": None, "tables": _ints(3, 5), "scale": -1.0}, "stored are"),
    ({"store": (torch.zeros(3, 128, dtype=BF16),) * 2, "tok_item": None, "tables": _ints(3, 5), "tok_list": _ints(3)}, "stored are"),
    ({"store": (torch.zeros(3, 128, dtype=BF16), torch.zeros(2, 128, dtype=BF16))}, "stored are")])
def test_decode_refused(on_gpu, changed, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.attention_decode_int4(**_decode(**changed))
    assert not on_gpu


@pytest.mark.parametrize("changed,message", [
    ({"q": torch.zeros(3, 256), "out": torch.zeros(3, 256)}, "bfloat16"), ({"heads": 3}, "do not fit"),
    ({"tile_q0": _ints(2)}, "inconsistent"), ({"cu_tokens": _ints(3)}, "inconsistent"), ({"tables": _ints(2, 5)}, "inconsistent"),
    ({"kv_lens": _ints(2)[::2]}, None), ({"kv_lens": _ints(4)[::2], "cu_tokens": _ints(3), "tables": _ints(2, 5)}, "contiguous"),
    ({"tile_item": _ints(1).long()}, "int32"), ({"sink": torch.zeros(5)}, "one float per head"),
    ({"ranges": 2, "query_tile": -64}, "queries"), ({"ranges": 2, "partial": torch.zeros(9, dtype=BF16)}, "partial"), ({"ranges": 2, "partial": torch.zeros(9, 2)[:, 0]}, "contiguous")])
def test_prompt_refused(on_gpu, changed, message):
    if message is None:
        kernels.attention_prefill_int4(**_prompt(**changed))
        return
    with pytest.raises(kernels.KernelError, match=message):
        kernels.attention_prefill_int4(**_prompt(**changed))
    assert not on_gpu


@pytest.mark.parametrize("changed,message", [
    ({"logits": torch.zeros(3, 50, dtype=torch.float16)}, "not supported"), ({"logits": torch.zeros(50, 3).t()}, "contiguous rows"),
    ({"tokens": _ints(2)}, "entry per row"), ({"tokens": _ints(3).long()}, "int32"), ({"out": torch.zeros(3, dtype=BF16)}, "float32"),
    ({"out": torch.zeros(6)[::2]}, "contiguous"), ({"entropy": torch.zeros(2)}, "entry per row"), ({"ranks": torch.zeros(3)}, "int32"),
    ({"top_ids": _ints(3, 4)}, "both or neither"), ({"top_ids": _ints(3, 4), "top_logprobs": torch.zeros(3, 5)}, "contiguous"),
    ({"top_ids": _ints(3, 33), "top_logprobs": torch.zeros(3, 33)}, "at most 32"),
    ({"logits": torch.zeros(3, 8), "top_ids": _ints(3, 9), "top_logprobs": torch.zeros(3, 9)}, "out of 8"),
    ({"top_ids": _ints(2, 4), "top_logprobs": torch.zeros(2, 4)}, "contiguous"), ({"partial": torch.zeros(4, dtype=BF16)}, "float32")])
def test_logprobs_refused(on_gpu, changed, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.token_logprobs(**_logprobs(**changed))
    assert not on_gpu


def _c(name, *args):
    lib = library.load_library()
    fn = getattr(lib, name)
    fn.argtypes, fn.restype = kernels._SIGNATURES[name], ctypes.c_int
    return fn(*args), lib.ps_last_error().decode()


ROWS = dict(table_width=5, tokens=3, kv_heads=2, head_dim=64, page_size=16, num_pages=4, dtype=0)


@pytest.mark.parametrize("name", ["ps_kv_write_int4", "ps_kv_read_int4"])
@pytest.mark.parametrize("changed,message", [
    ({"tokens": -1}, "bad sizes"), ({"table_width": 0}, "bad sizes"), ({"head_dim": 257}, "1..256"), ({"head_dim": 0}, "1..256"),
    ({"page_size": 12}, "multiple of 8"), ({"dtype": 2}, "dtype"), ({"kv_heads": 3}, "stride"), ({"num_pages": 0}, "bad sizes")])
def test_rows_refused_by_the_library(name, changed, message):
    sizes = dict(ROWS, **changed)
    status, error = _c(name, 0, 0, 0, 0, 128, 128, 0, 0, 0, *sizes.values(), 0) if name.endswith("read_int4") \
        else _c(name, 0, 0, 128, 128, 0, 0, 0, 0, 0, *sizes.values(), 0)
    assert status == 1 and message in error and name in error


ATTEND = dict(table_width=5, count=3, heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, scale=0.125, window=0, splits=1)


@pytest.mark.parametrize("changed,message", [
    ({"heads": 5}, "multiple of kv_heads"), ({"head_dim": 257}, "1..256"), ({"page_size": 20}, "multiple of 8"),
    ({"splits": 65}, "64 ranges"), ({"splits": 0}, "64 ranges"), ({"splits": 2}, "too few"), ({"count": -1}, "bad sizes"),
    ({"table_width": 1 << 26}, "block tables")])
def test_decode_refused_by_the_library(changed, message):
    sizes = dict(ATTEND, **changed)
    status, error = _c("ps_attention_decode_int4", 0, 256, 0, 0, 0, 0, 0, 0, 0, 256, 0, 0, 0, 0, 0, 0, *sizes.values(), 0, 0.0, 1, 0)
    assert status == 1 and message in error


PORTIONS = dict(table_width=5, heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, scale=0.125, window=0, max_kv_len=0,
                query_tile=64, sink=0, softcap=0.0, block_heads=1, ranges=1)


@pytest.mark.parametrize("changed,message", [
    ({"heads": 5}, "multiple of kv_heads"), ({"head_dim": 72}, "multiple of 16"), ({"head_dim": 272}, "up to 256"),
    ({"page_size": 20}, "multiple of 8"), ({"query_tile": 96}, "queries"), ({"query_tile": 128, "head_dim": 144}, "queries"), ({"block_heads": 2, "head_dim": 64}, "heads to a block"),
    ({"block_heads": 2, "head_dim": 144}, "heads to a block"), ({"block_heads": 2, "head_dim": 128, "query_tile": 128}, "heads to a block"),
    ({"block_heads": 2, "head_dim": 128, "heads": 6}, "heads to a block"), ({"block_heads": 3}, "heads to a block"),
    ({"query_tile": 32}, "queries"), ({"ranges": 0}, "ranges"), ({"ranges": 65}, "ranges"), ({"ranges": 2}, "floats of scratch"), ({"scale": 0.0}, "positive"), ({"table_width": 2049}, "exceed"),
    ({"num_pages": 1 << 28}, "key rows")])
def test_prompt_refused_by_the_library(changed, message):
    sizes = dict(PORTIONS, **changed)
    status, error = _c("ps_attention_prefill_int4", 0, 256, 0, 0, 0, 256, 0, 0, 1, 0, 0, 0, *sizes.values(), 0, 0, 0)
    assert status == 1 and message in error
    status, error = _c("ps_attention_prefill_int4", 0, 252, 0, 0, 0, 256, 0, 0, 1, 0, 0, 0, *PORTIONS.values(), 0, 0, 0)
    assert status == 1 and "accesses" in error


@pytest.mark.parametrize("changed,message", [
    ({"q": torch.zeros(3, 256, dtype=BF16), "out": torch.zeros(3, 256, dtype=BF16)}, "float32"), ({"heads": 3}, "do not fit"),
    ({"out": torch.zeros(3, 128)}, "rows must hold"), ({"tile_q0": _ints(2)}, "inconsistent"), ({"cu_tokens": _ints(3)}, "inconsistent"),
    ({"tables": _ints(2, 5)}, "inconsistent"), ({"kv_lens": _ints(4)[::2], "cu_tokens": _ints(3), "tables": _ints(2, 5)}, "contiguous"),
    ({"tile_item": _ints(1).long()}, "int32"), ({"sink": torch.zeros(5)}, "one float per head"), ({"softcap": -1.0}, "score cap")])
def test_float_prompt_refused(on_gpu, changed, message):
    with pytest.raises(kernels.KernelError, match=message):
        kernels.attention_tiled_f32_int4(**_float_prompt(**changed))
    assert not on_gpu


FLOATS = dict(table_width=5, heads=4, kv_heads=2, head_dim=64, page_size=16, num_pages=4, scale=0.125, window=0, sink=0, softcap=0.0,
              query_tile=64, paired=0)


@pytest.mark.parametrize("changed,message", [
    ({"heads": 5}, "multiple of kv_heads"), ({"head_dim": 66}, "multiple of 4"), ({"head_dim": 132}, "up to 128"),
    ({"page_size": 20}, "multiple of 8"), ({"query_tile": 128}, "queries"), ({"query_tile": 32, "paired": 1}, "queries"),
    ({"scale": 0.0}, "positive"), ({"table_width": 0}, "bad sizes")])
def test_float_prompt_refused_by_the_library(changed, message):
    sizes = dict(FLOATS, **changed)
    status, error = _c("ps_attention_tiled_f32_int4", 0, 256, 0, 0, 0, 256, 0, 0, 1, 0, 0, 0, *sizes.values(), 0)
    assert status == 1 and message in error
    status, error = _c("ps_attention_tiled_f32_int4", 0, 254, 0, 0, 0, 256, 0, 0, 1, 0, 0, 0, *FLOATS.values(), 0)
    assert status == 1 and "accesses" in error
    assert _c("ps_attention_tiled_f32_int4", 0, 256, 0, 0, 0, 256, 0, 0, 0, 0, 0, 0, *FLOATS.values(), 0)[0] == 0


@pytest.mark.parametrize("args,message", [
    ((49, 3, 50, 0), "bad sizes"), ((50, -1, 50, 0), "bad sizes"), ((50, 3, 50, 33), "alternatives"), ((50, 3, 8, 9), "alternatives"),
    ((1 << 30, 3, 1 << 30, 0), "too large"), ((200000, 1, 200000, 0), "too few")])
def test_logprobs_refused_by_the_library(args, message):
    ld, rows, vocab, top = args
    status, error = _c("ps_token_logprobs", 0, ld, rows, vocab, 0, 0, 0, 0, 0, 0, top, 0, 0, 0, 0)
    assert status == 1 and message in error


def test_nothing_to_do_is_no_launch():
    """No tokens, no rows, no tiles: success before anything is launched."""
    sizes = dict(ROWS, tokens=0)
    assert _c("ps_kv_write_int4", 0, 0, 128, 128, 0, 0, 0, 0, 0, *sizes.values(), 0)[0] == 0
    assert _c("ps_token_logprobs", 0, 50, 0, 50, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)[0] == 0
    sizes = dict(ATTEND, count=0)
    assert _c("ps_attention_decode_int4", 0, 256, 0, 0, 0, 0, 0, 0, 0, 256, 0, 0, 0, 0, 0, 0, *sizes.values(), 0, 0.0, 1, 0)[0] == 0
    assert _c("ps_attention_prefill_int4", 0, 256, 0, 0, 0, 256, 0, 0, 0, 0, 0, 0, *PORTIONS.values(), 0, 0, 0)[0] == 0


@pytest.mark.parametrize("dim", [1, 7, 32, 33, 64, 250])
def test_the_form_itself(dim):
    """Every value that the cache can hold is a bfloat16 number, the largest one is held to its step's rounding, and no
    element is off by more than half a step (one and a quarter on the side that has seven codes)."""
    g = torch.Generator().manual_seed(dim)
    rows = torch.randn((40, 2 * dim), generator=g) * torch.logspace(-3, 3, 40)[:, None]
    codes, steps, values = plain.held(rows, 2)
    assert torch.equal(values.to(BF16).double(), values)
    assert codes.min() >= 0 and codes.max() <= 15
    groups = steps.shape[2]
    per = torch.from_numpy(abs(steps)).repeat_interleave(32, dim=2)[..., :dim].reshape(40, 2 * dim)
    off = (values - rows.double()).abs()
    assert bool((off <= 1.26 * per).all()) and groups == -(-dim // 32)
    assert float((off <= 0.51 * per).double().mean()) > 0.9
    assert kernels.int4_row_bytes(dim) == 18 * groups


@pytest.mark.skipif(kernel_code.disassembler() is None, reason="no disassembler")
@pytest.mark.parametrize("kernel", ["attention_prefill_int4_kernel", "attention_decode_int4_heads_kernel"])
def test_no_register_is_used_before_its_load(kernel, tmp_path):
    """Every instance of the kernels that read their operands from LDS by assembly, as built."""
    path = os.path.join(library.in_tree_dir(), library.LIB_NAME)
    if not os.path.isfile(path):
        pytest.skip("the library is not built in the tree")
    images = [image for image in kernel_code.code_objects(path, library.ARCH) if kernel.encode() in image]
    assert images, "no source file holds this kernel"
    seen = 0
    for image in images:
        for name, code in kernel_code.kernels(kernel_code.disassemble(image, library.ARCH, tmp_path)):
            if kernel in name:
                seen += 1
                assert any(operation.startswith("ds_read") for _, operation, _, _ in code), name
                assert not kernel_code.early_uses(code), (name, kernel_code.early_uses(code)[:4])
    assert seen > 3

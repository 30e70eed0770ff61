"""Sizes beyond what a call takes are wrong arguments like others: ValueError, nothing launched."""
import pytest
import torch

import okc_muse_kernels_b200 as okc
from okc_muse_kernels_b200 import _lib


@pytest.mark.parametrize("rows", [(1 << 30) + 1, (1 << 31) + 5])
def test_more_tokens_or_outputs_than_the_products_take(rows):
    """(meta tensors: sizes without memory)"""
    few, many = torch.empty((2, 16), dtype=torch.bfloat16, device="meta"), torch.empty((rows, 16), dtype=torch.bfloat16, device="meta")
    def quant(r):
        return torch.empty((r, 16), dtype=torch.int8, device="meta"), torch.empty(r, device="meta")
    for fn, per in ((okc.int8_linear, 1), (okc.int8_gated, 2)):
        for x in (many, quant(rows)):
            with pytest.raises(ValueError, match="at most"):
                fn(x, quant(2))
        with pytest.raises(ValueError, match="at most"):
            fn(few, quant(rows * per))


def test_more_rows_than_a_call_takes():
    x = torch.empty((1 << 31, 8), dtype=torch.bfloat16, device="meta")
    for call in (lambda: okc.quantize_rows(x), lambda: okc.block_norm(x, x), lambda: okc.block_norm(x, pre_gain=torch.empty(8, device="meta"))):
        with pytest.raises(ValueError, match="at most"):
            call()


def test_scratch_of_no_tokens():
    need = _lib.lib().okc_moe_int8_scratch_bytes
    assert need(0, 0, 4096) == 0 and need(0, -1, 4096) == 0 and need(1, -(1 << 31), 16) == 0 and need(0, 5, 0) == 0 and need(0, 5, -7) == 0
    assert need(0, 1 << 30, 131071) == (1 << 30) * (131072 + 4)

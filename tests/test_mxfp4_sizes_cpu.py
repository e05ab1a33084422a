"""Sizes beyond the C ABI's int32: refused, not cut (no GPU and no memory needed: the rows of
these tensors are one row)."""

from __future__ import annotations

import pytest
import torch

from int8_linear import NotSupported, _native, mxfp4
from int8_linear.qk_norm import qk_norm_rope

MANY = 2 ** 32 + 128


def rows(n, cols, dtype):
    return torch.zeros((1, cols), dtype=dtype).expand(n, cols)


@pytest.mark.parametrize("n", [2 ** 31, MANY])
def test_more_rows_than_int32_holds(n):
    x, q = rows(n, 64, torch.bfloat16), rows(n, 32, torch.uint8)
    s = torch.zeros((1, 1, 512), dtype=torch.uint8)
    many_s = s.expand(-(-n // 128), 1, 512)
    one = torch.ones(64)
    small = torch.zeros((1, 32), dtype=torch.uint8)
    for call in (lambda: mxfp4.quant_mxfp4(x), lambda: mxfp4.silu_mul_quant_mxfp4(x),
                 lambda: mxfp4.add_rmsnorm_quant_mxfp4(x, None, one, 1e-6), lambda: mxfp4.dequant_mxfp4(q, many_s),
                 lambda: mxfp4.w4a4_mm(small, q.t(), s, many_s), lambda: mxfp4.w4a4_mm(q, small.t(), many_s, s),
                 lambda: qk_norm_rope(x, one[:32], one[:32], 1e-6, torch.zeros(1, dtype=torch.int64).expand(n),
                                      torch.zeros((1, 32)), 1, 1)):
        with pytest.raises(NotSupported):
            call()

def test_norm_whose_grid_would_be_too_large():
    p = 1 << 20   # never dereferenced: refused before any CUDA call
    lib = _native.load()
    assert lib.i8l_add_rmsnorm_quant_mxfp4(p, 32, None, 0, p, 0, 0, p, 16, p, None, 0, 2 ** 31 - 1, 32, 1e-6,
                                           None) == _native.ENOTSUP

def test_meta_function_of_the_norm_has_the_strides_of_the_op():
    x = torch.empty((64, 48), dtype=torch.bfloat16, device="meta").t()
    q, s, res = torch.ops.int8_linear.add_rmsnorm_quant_mxfp4(x, x, torch.empty(64, device="meta"), 1e-6)
    assert res.shape == (48, 64) and res.is_contiguous()

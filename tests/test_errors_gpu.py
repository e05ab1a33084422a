"""A call that failed is reported once: the thread's next call is not affected."""

from __future__ import annotations

import pytest
import torch

from int8_linear import _native, mxfp4
from int8_linear.fused_quant import per_token_quant
from int8_linear.qk_norm import qk_norm_rope

pytestmark = pytest.mark.gpu


def test_the_call_after_a_failed_one_succeeds():
    x = torch.ones((3, 128), dtype=torch.bfloat16, device="cuda")
    ones, cs = torch.ones(64, device="cuda"), torch.ones((1, 64), device="cuda")
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    q, s = mxfp4.quant_mxfp4(x)
    w = x.new_ones((64, 128))
    wq, ws = mxfp4.quant_mxfp4(w)
    calls = [lambda: mxfp4.quant_mxfp4(x), lambda: mxfp4.w4a4_mm(q, wq.t(), s, ws), lambda: per_token_quant(x),
             lambda: qk_norm_rope(x, ones, ones, 1e-6, pos, cs, 1, 1), lambda: mxfp4.dequant_mxfp4(q, s),
             lambda: mxfp4.silu_mul_quant_mxfp4(x), lambda: mxfp4.add_rmsnorm_quant_mxfp4(x, x, x[0], 1e-6)]
    host = torch.zeros(4)
    for call in calls:
        with pytest.raises(RuntimeError):   # the runtime refuses to free memory that is not its own
            _native.check(_native.load().i8l_peer_free(host.data_ptr()))
        call()
    torch.cuda.synchronize()

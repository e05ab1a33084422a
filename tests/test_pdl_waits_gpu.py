"""Products launched programmatically behind a kernel that runs longer than their own waits
may last: the limit of a wait counts from when that kernel is done.

The long kernel is a tensor-parallel exchange whose peer never signals; it gives up after
three seconds, a product's waits after two."""

from __future__ import annotations

import ctypes

import pytest
import torch

import int8_linear
from int8_linear import Config, _native, mxfp4, w8a8_mm
from tests.gpu_util import ints, rand
from tests.test_peer_gpu import PEER_WAIT_BIT, _lonely_comm

pytestmark = pytest.mark.gpu


def four(m, cfg):
    def make():
        a, sa = mxfp4.quant_mxfp4(rand((m, 4096), 1))
        w, sw = mxfp4.quant_mxfp4(rand((512, 4096), 2))
        return lambda: mxfp4.w4a4_mm(a, w.t(), sa, sw, torch.float32, config=cfg)
    return make


def eight(m, cfg):
    def make():
        a, w, one = ints((m, 4096), 1), ints((512, 4096), 2), torch.ones(1, device="cuda")
        return lambda: w8a8_mm(a, w.t(), one, one, torch.float32, config=cfg)
    return make


@pytest.mark.parametrize("make", [four(16, Config(16, 128, swap_ab=True, split=3, cluster=2)),
                                  four(300, Config(128, 256, split=4)), four(2, Config(2, 0, split=5)),
                                  eight(300, Config(128, 128)), eight(300, Config(128, 256, split=4)),
                                  eight(2, Config(2, 0, stages=1, ctas=8, split=5))],
                         ids=["split", "pair", "CUDA cores", "int8", "int8 pair", "int8 CUDA cores"])
def test_product_behind_a_long_kernel(make):
    lib = _native.load()
    _native.clear_status()
    call = make()
    want = call()
    d, own, epochs = _lonely_comm(timeout_ns=3_000_000_000)
    x = rand((1, 256), 3)
    q = torch.empty((1, 256), dtype=torch.int8, device="cuda")
    s = torch.empty((1, 1), dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    int8_linear.set_pdl(True)
    try:
        _native.check(lib.i8l_tp_quant_rows(ctypes.byref(d), x.data_ptr(), 256, _native.BF16, q.data_ptr(), 256,
                                            s.data_ptr(), 1, 256, 1, torch.cuda.current_stream().cuda_stream))
        got = call()
    finally:
        int8_linear.set_pdl(False)
    assert _native.read_status() == PEER_WAIT_BIT
    _native.clear_status()
    assert torch.equal(got, want)
    _native.check(lib.i8l_peer_free(own))

"""Weights quantised in the same stream as the products that read them, under programmatic
dependent launch: a product loads its weight before it waits for the kernels before it."""

from __future__ import annotations

import pytest
import torch

import int8_linear
from int8_linear import Config, _native, mxfp4
from int8_linear.fused_quant import add_rmsnorm_quant
from tests.gpu_util import rand

pytestmark = pytest.mark.gpu


@pytest.fixture
def pdl():
    before = int8_linear.pdl_enabled()
    int8_linear.set_pdl(True)
    yield
    int8_linear.set_pdl(before)


@pytest.mark.parametrize("between", ["nothing", "one", "several"])
@pytest.mark.parametrize("m,n,k,cfg", [(2, 4096, 2048, Config(4, 0, split=5)), (16, 8192, 8192, None),
                                       (100, 8192, 4096, Config(128, 128, swap_ab=True, split=1)),
                                       (600, 4096, 8192, Config(128, 256, split=4)), (2, 128, 256, Config(4, 0, split=5)),
                                       (2, 127, 4096, Config(4, 0, split=5)), (16, 100, 16384, None),
                                       (300, 127, 8192, Config(128, 256, split=4))])
def test_weight_quantised_just_before_its_product(m, n, k, cfg, between, pdl):
    """The weight's buffers hold another weight's codes from the turn before (the allocator
    hands them out again), so that a product that reads them too early differs."""
    x, gamma = rand((m, k), 1), rand((k,), 2, 0.1) + 1
    weights = [rand((n, k), 3 + i, dtype=t) for i, t in enumerate((torch.bfloat16, torch.float32))]
    small = rand((3, 256), 9)

    def turn(w):
        q, s = mxfp4.quant_mxfp4(x)
        torch.cuda.synchronize()
        b, sb = mxfp4.quant_mxfp4(w)
        if between != "nothing":
            q, s, _ = mxfp4.add_rmsnorm_quant_mxfp4(x, None, gamma, 1e-6)
        if between == "several":
            for _ in range(3):
                add_rmsnorm_quant(small, None, gamma[:256], 1e-6)
        return mxfp4.w4a4_mm(q, b.t(), s, sb, torch.float32, config=cfg)

    int8_linear.set_pdl(False)
    want = [turn(w) for w in weights]
    int8_linear.set_pdl(True)
    for _ in range(10):
        for w, y in zip(weights, want):
            assert torch.equal(turn(w), y)
    graphs = []
    for w in weights:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            b, sb = mxfp4.quant_mxfp4(w)
            q, s, _ = mxfp4.add_rmsnorm_quant_mxfp4(x, None, gamma, 1e-6)
            graphs.append((g, mxfp4.w4a4_mm(q, b.t(), s, sb, torch.float32, config=cfg)))
    int8_linear.set_pdl(False)
    for w, (g, got) in zip(weights, graphs):
        b, sb = mxfp4.quant_mxfp4(w)
        q, s, _ = mxfp4.add_rmsnorm_quant_mxfp4(x, None, gamma, 1e-6)
        y = mxfp4.w4a4_mm(q, b.t(), s, sb, torch.float32, config=cfg)
        for _ in range(3):
            g.replay()
            assert torch.equal(got, y)
    assert _native.read_status() == 0

"""A product as the first CUDA call of a host thread."""

from __future__ import annotations

import threading

import pytest
import torch

from int8_linear import Config, mxfp4, w8a8_mm
from tests.gpu_util import ints

pytestmark = pytest.mark.gpu


def in_new_thread(call):
    got = []

    def run():
        try:
            got.append(call())
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("m", [1, 16, 300])
def test_int8_product(m):
    a, w = ints((m, 512), 1), ints((256, 512), 2)
    one = torch.ones(1, device="cuda")
    for cfg in (None, Config(128, 128)):
        want = w8a8_mm(a, w.t(), one, one, torch.float32, config=cfg)
        torch.cuda.synchronize()
        assert torch.equal(in_new_thread(lambda: w8a8_mm(a, w.t(), one, one, torch.float32, config=cfg)), want)


@pytest.mark.parametrize("m", [1, 16, 300])
def test_4_bit_product(m):
    a, sa = mxfp4.quant_mxfp4(torch.randn((m, 512), device="cuda"))
    w, sw = mxfp4.quant_mxfp4(torch.randn((256, 512), device="cuda"))
    for cfg in (None, Config(128, 128, swap_ab=True, split=1), Config(128, 256, split=4)):
        want = mxfp4.w4a4_mm(a, w.t(), sa, sw, config=cfg)
        torch.cuda.synchronize()
        assert torch.equal(in_new_thread(lambda: mxfp4.w4a4_mm(a, w.t(), sa, sw, config=cfg)), want)

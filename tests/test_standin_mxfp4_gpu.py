"""The 4-bit operators together, as the decoder runs them: every op of a step on its own
inputs against the oracle, the step's chaining, and captured steps that are replayed with
other inputs, with and without programmatic dependent launch."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8_linear
from int8_linear import _native
from int8_linear.standin import (EPS, HEAD_DIM, HIDDEN, KV_HEADS, LAYERS, Q_HEADS, SHAPES, MXFP4StandinDecoder)
from oracle import mxfp4 as om
from oracle.numerics import to_bits
from tests.gpu_util import bits, np_
from tests.test_qk_norm_gpu import check as check_qk

pytestmark = pytest.mark.gpu


def check_codes(q, s, y):
    codes, e = om.quantise(y)
    assert np.array_equal(np_(q), om.pack(codes)) and np.array_equal(np_(s), om.tile_scales(e))


def check_mm(q, s, lin, out):
    """Within K roundings of float32 of the exact product and half a step of bf16."""
    a = torch.from_numpy(om.operand_values(np_(q), np_(s))).cuda()
    w = torch.from_numpy(om.operand_values(np_(lin.q_t.t()), np_(lin.scale))).cuda()
    want, size = a @ w.t(), (a.abs() @ w.abs().t()) * (a.shape[1] * 2.0 ** -23)
    info = torch.finfo(torch.bfloat16)
    err = (out.double() - want).abs()
    assert (err <= size + (want.abs() + size) * info.eps / 2 + info.tiny).all()


@pytest.mark.parametrize("m", [1, 5, 64, 130])
def test_every_op_of_a_step(m):
    dec = MXFP4StandinDecoder(m, layers=2)
    record: list = []
    out = dec.step(record)
    assert out.shape == (m, HIDDEN) and torch.isfinite(out).all()
    assert [name for i, name, _, _ in record if i == 1] == [
        "norm", "qkv_proj", "qk_norm", "quant", "o_proj", "post_norm", "gate_up_proj", "silu_mul_quant", "down_proj"]
    for _, name, ins, outs in record:
        if name in SHAPES:
            check_mm(*ins, outs)
        elif name in ("norm", "post_norm"):
            x, res, w = ins
            y, r = om.norm_rows(np_(x), None if res is None else np_(res), np_(w), EPS, "bf16", "bf16")
            check_codes(outs[0], outs[1], y)
            if res is not None:
                assert np.array_equal(bits(outs[2]), to_bits(r, "bf16"))
        elif name == "qk_norm":
            qkv, wq, wk, pos, cs = ins
            check_qk(qkv, wq, wk, pos, cs, Q_HEADS, KV_HEADS, False, outs)
        elif name == "quant":
            check_codes(*outs, np_(ins[0]))
        else:
            check_codes(*outs, om.silu_rows(np_(ins[0]), "bf16"))
    # each op's input is the op before's output
    by = {(i, name): (ins, outs) for i, name, ins, outs in record}
    for i in range(2):
        assert by[i, "qkv_proj"][0][0] is by[i, "norm"][1][0]
        assert by[i, "qk_norm"][0][0] is by[i, "qkv_proj"][1]
        assert by[i, "quant"][0][0].data_ptr() == by[i, "qk_norm"][1][0].data_ptr()
        assert by[i, "post_norm"][0][0] is by[i, "o_proj"][1]
        assert by[i, "silu_mul_quant"][0][0] is by[i, "gate_up_proj"][1]
        assert by[i, "down_proj"][0][0] is by[i, "silu_mul_quant"][1][0]
    assert by[1, "norm"][0][0] is by[0, "down_proj"][1] and by[1, "norm"][0][1] is by[0, "post_norm"][1][2]
    assert by[0, "post_norm"][0][1] is dec.x and out is by[1, "down_proj"][1]
    assert _native.read_status() == 0


@pytest.mark.parametrize("m", [1, 33, 300])
@pytest.mark.parametrize("pdl", [False, True])
def test_captured_steps_replay_with_other_inputs(m, pdl):
    was = int8_linear.pdl_enabled()
    int8_linear.set_pdl(pdl)
    try:
        dec = MXFP4StandinDecoder(m, layers=3)
        dec.capture()
        for seed in (1, 2):
            g = torch.Generator(device="cuda").manual_seed(seed)
            dec.x.copy_(torch.randn((m, HIDDEN), generator=g, device="cuda"))
            dec.positions.copy_(torch.randint(0, 4096, (m,), generator=g, device="cuda"))
            for _ in range(3):
                dec.graph.replay()
            got = dec.out.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, dec.step())
        assert _native.read_status() == 0
    finally:
        int8_linear.set_pdl(was)


def test_weights_take_a_quarter_of_bf16():
    dec = MXFP4StandinDecoder(1, layers=1)
    values = sum(k * n for k, n in SHAPES.values())
    assert dec.weight_bytes() == values // 2 + values // 32 and LAYERS == 28 and Q_HEADS * HEAD_DIM == HIDDEN

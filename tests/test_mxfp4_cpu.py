"""Refusals of the 4-bit and query/key entry points that need no GPU, and the oracle's own
layout helpers."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int8_linear import NotSupported, _native, mxfp4
from int8_linear.qk_norm import qk_norm_rope
from oracle import mxfp4 as om


def test_oracle_tiles_and_packing_round_trip():
    rng = np.random.default_rng(0)
    for r, nb in ((1, 1), (33, 5), (129, 4), (300, 9)):
        s = rng.integers(0, 255, (r, nb)).astype(np.uint8)
        t = om.tile_scales(s)
        assert t.shape == (-(-r // 128), -(-nb // 4), 512) and np.array_equal(om.untile_scales(t, r, nb), s)
    c = rng.integers(0, 16, (7, 64)).astype(np.uint8)
    assert np.array_equal(om.unpack(om.pack(c)), c)


def test_oracle_rounds_to_the_nearest_value():
    """Against a search over all sixteen values of each block's grid."""
    rng = np.random.default_rng(1)
    y = (rng.standard_normal((8, 64)) * np.exp2(rng.integers(-5, 5, (8, 64)))).astype(np.float32)
    codes, s = om.quantise(y)
    v = om.values(codes, s)
    grid = np.concatenate([om.GRID, -om.GRID])
    scale = np.repeat(np.exp2(s.astype(np.float64) - 127), 32, axis=1)
    best = np.abs(grid[:, None, None] * scale - y.astype(np.float64)).min(0)
    assert np.array_equal(np.abs(v - y.astype(np.float64)), best)


def test_c_refusals_come_before_any_cuda_call():
    lib = _native.load()
    ok, notsup, inval = _native.OK, _native.ENOTSUP, _native.EINVAL
    p = 1 << 20                                   # never dereferenced: every call is refused
    assert lib.i8l_quant_mxfp4(p, 64, 7, p, 32, p, 2, 64, None) == notsup
    assert lib.i8l_quant_mxfp4(p, 64, 0, p, 32, p, 2, 48, None) == notsup
    assert lib.i8l_quant_mxfp4(p, 64, 0, p, 32, p, -1, 64, None) == inval
    assert lib.i8l_quant_mxfp4(p, 63, 0, p, 32, p, 2, 64, None) == inval
    assert lib.i8l_quant_mxfp4(p, 64, 0, p, 31, p, 2, 64, None) == inval
    assert lib.i8l_quant_mxfp4(p, 64, 0, p + 1, 32, p, 2, 64, None) == notsup
    assert lib.i8l_quant_mxfp4(None, 64, 0, p, 32, p, 2, 64, None) == inval
    assert lib.i8l_quant_mxfp4(p, 1 << 27, 0, p, 1 << 26, p, 2, 1 << 27, None) == notsup
    assert lib.i8l_quant_mxfp4(None, 64, 0, None, 32, None, 0, 64, None) == ok
    assert lib.i8l_silu_mul_quant_mxfp4(p, 64, 2, p, 32, p, 2, 64, None) == notsup
    assert lib.i8l_silu_mul_quant_mxfp4(p, 127, 0, p, 32, p, 2, 64, None) == inval
    assert lib.i8l_add_rmsnorm_quant_mxfp4(p, 64, p, 64, p, 0, 0, p, 32, p, None, 64, 2, 64, 1e-6, None) == inval
    assert lib.i8l_add_rmsnorm_quant_mxfp4(p, 64, None, 0, p, 0, 5, p, 32, p, None, 0, 2, 64, 1e-6, None) == notsup
    assert lib.i8l_add_rmsnorm_quant_mxfp4(p, 65536, None, 0, p, 0, 0, p, 32768, p, None, 0, 2, 65536, 1e-6,
                                           None) == notsup
    assert lib.i8l_dequant_mxfp4(p, 32, p, p, 63, 0, 2, 64, None) == inval
    assert lib.i8l_dequant_mxfp4(p, 32, p, p, 64, 3, 2, 64, None) == notsup
    assert lib.i8l_mxfp4_scale_bytes(129, 160) == 2 * 2 * 512 and lib.i8l_mxfp4_scale_bytes(0, 64) == 0

    def mm(m=4, n=8, k=64, lda=32, ldw=32, ldc=8, a=p, sw=p, bias=None, bdt=0, odt=0, out=p):
        return lib.i8l_w4a4_mm(a, lda, p, p, ldw, sw, bias, bdt, out, odt, ldc, m, n, k, None, None)

    assert mm(odt=3) == notsup and mm(k=48) == notsup and mm(k=0) == notsup and mm(bias=p, bdt=3) == notsup
    assert mm(m=-1) == inval and mm(lda=16) == inval and mm(ldw=16) == inval and mm(ldc=7) == inval
    assert mm(a=None) == inval and mm(sw=None) == inval and mm(out=None) == inval
    assert mm(a=p + 8) == notsup and mm(sw=p + 4) == notsup and mm(lda=40) == notsup
    assert mm(n=2 ** 31 - 1, ldc=2 ** 31) == notsup and mm(m=0) == ok and mm(n=0) == ok

    def qk(ld=512, act=0, dim=64, rot=64, inter=0, tokens=2, heads=4, kv=2, qkv=p, ldq=256, ldk=128, cs=p):
        return lib.i8l_qk_norm_rope(qkv, ld, act, p, p, 0, 1e-6, p, 1, cs, 2, 10, p, ldq, p, ldk, tokens, heads,
                                    kv, dim, rot, inter, None)

    assert qk(act=2) == notsup and qk(dim=60) == inval and qk(dim=60, rot=48) == notsup and qk(dim=264, rot=0) == notsup
    assert qk(rot=24) == notsup and qk(rot=4, inter=1) == notsup and qk(rot=72) == inval
    assert qk(ld=383) == inval and qk(ldq=255) == inval and qk(ldk=127) == inval and qk(cs=None) == inval
    assert qk(ld=516) == notsup and qk(qkv=p + 2) == notsup and qk(ldk=132) == notsup
    assert qk(tokens=0) == ok and qk(heads=0, kv=0) == ok and qk(tokens=-1) == inval


def test_python_refuses_cpu_tensors_and_bad_types():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    w = torch.zeros(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        mxfp4.quant_mxfp4(x)
    with pytest.raises(NotSupported):
        mxfp4.quant_mxfp4(x.to(torch.int8))
    with pytest.raises(ValueError):
        mxfp4.silu_mul_quant_mxfp4(x)
    with pytest.raises(ValueError):
        mxfp4.dequant_mxfp4(torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8))
    q, s = torch.zeros((2, 32), dtype=torch.uint8), torch.zeros((1, 1, 512), dtype=torch.uint8)
    with pytest.raises(ValueError):
        mxfp4.w4a4_mm(q, q.t(), s, s)
    with pytest.raises(ValueError):
        mxfp4.add_rmsnorm_quant_mxfp4(x, None, w, 1e-6)
    with pytest.raises(ValueError):
        qk_norm_rope(x, w, w, 1e-6, torch.zeros(2, dtype=torch.int64), torch.zeros((4, 64)), 1, 0)

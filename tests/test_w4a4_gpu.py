"""The 4-bit product (w4a4_mm) against float64.

Two kinds of operands.  With few scales, every product is a multiple of 2^-4 and every sum
stays below 2^19, so float32 holds each partial sum exactly and the float32 output has to
equal the exact product in every bit, whatever the order of the additions.  With scales of
any size, a sum of K products in float32 is off by at most K * 2^-23 of the sum of their
magnitudes (K additions, each losing less than one unit in the last place of 24 bits), plus
half a step of the output's type.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import int8_linear
from int8_linear import Config, NotSupported, _native, mxfp4
from oracle import mxfp4 as om
from tests.gpu_util import np_, rand

pytestmark = pytest.mark.gpu


def operand(rows, k, seed, spread=1, nan_pad=False):
    """Random codes and scale bytes 127 - spread .. 127 + spread: (q, s, float64 values) on
    the GPU.  nan_pad: the scale bytes of rows past the last hold 0xFF."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    e = torch.randint(127 - spread, 128 + spread, (rows, k // 32), generator=g, dtype=torch.uint8)
    tiles = om.tile_scales(e.numpy())
    if nan_pad and rows % 128:
        full = om.tile_scales(np.full((tiles.shape[0] * 128 - rows + rows, k // 32), 255, np.uint8))
        keep = om.tile_scales(np.ones((rows, k // 32), np.uint8)) > 0
        tiles = np.where(keep, tiles, full)
    q, s = q.cuda(), torch.from_numpy(tiles).cuda()
    return q, s, torch.from_numpy(om.operand_values(q.cpu().numpy(), tiles)).cuda()


def exact(m, n, k, cfg=None, seed=0, **kw):
    a, sa, va = operand(m, k, 10 + seed, **kw)
    b, sb, vb = operand(n, k, 20 + seed, **kw)
    assert (va.abs() @ vb.abs().t()).max().item() < 2.0 ** 19
    got = mxfp4.w4a4_mm(a, b.t(), sa, sb, torch.float32, config=cfg)
    want = va @ vb.t()
    assert torch.equal(got.double(), want), (got.double() - want).abs().max()
    assert _native.read_status() == 0


@pytest.mark.parametrize("m,n,k", [(1, 128, 256), (1, 1, 32), (3, 130, 64), (16, 128, 96), (16, 256, 2048),
                                   (17, 100, 160), (33, 515, 544), (64, 384, 1024), (65, 96, 224), (128, 128, 512),
                                   (129, 257, 288), (300, 640, 2080), (1, 4096, 2048), (8, 2048, 6144),
                                   (1000, 300, 768)])
def test_sums_that_float32_holds_exactly(m, n, k):
    exact(m, n, k)


@pytest.mark.parametrize("tn", [16, 32, 64, 128])
@pytest.mark.parametrize("cluster", [1, 2, 3, 5, 8])
@pytest.mark.parametrize("stages", [0, 1, 2])
def test_every_split_tile(tn, cluster, stages):
    cfg = Config(tn, 128, swap_ab=True, split=3 if cluster > 1 else 1, cluster=cluster, stages=stages)
    exact(min(tn, 61), 200, 2336, cfg, seed=cluster)
    if tn == 128:
        exact(200, 200, 2336, cfg, seed=cluster)


@pytest.mark.parametrize("m", [1, 2, 3, 4])
@pytest.mark.parametrize("n,k", [(1, 32), (33, 96), (130, 160), (257, 2048), (515, 2080), (100, 4128), (4096, 2048),
                                 (12300, 544)])
def test_cuda_core_tiles(m, n, k):
    exact(m, n, k, Config(4 if m == 3 else m, 0, split=5), seed=m)


@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (128, 256, 256), (256, 256, 64), (257, 513, 1056), (300, 40, 2336),
                                   (1000, 1000, 992), (2600, 3000, 288)])
@pytest.mark.parametrize("stages,ctas", [(0, 0), (2, 0), (3, 6)])
def test_pair_tiles(m, n, k, stages, ctas):
    """Few pairs make each one walk over many tiles, through both accumulators."""
    exact(m, n, k, Config(128, 256, split=4, stages=stages, ctas=ctas))


def test_scale_bytes_of_no_row_do_not_matter():
    exact(5, 130, 160, nan_pad=True)
    exact(140, 130, 160, nan_pad=True)


def near(a, sa, va, b, sb, vb, dtype, bias=None, cfg=None, out=None):
    got = mxfp4.w4a4_mm(a, b.t(), sa, sb, dtype, bias, config=cfg, out=out)
    k = va.shape[1]
    want = va @ vb.t()
    size = (va.abs() @ vb.abs().t()) * k * 2.0 ** -23
    if bias is not None:
        want = want + bias.double()
        size = size + want.abs() * 2.0 ** -23
    info = torch.finfo(dtype)
    tol = size + (want.abs() + size) * info.eps / 2 + info.tiny * info.eps / 2
    err = (got.double() - want).abs()
    assert got.dtype == dtype and (err <= tol).all(), (err - tol).max()
    assert _native.read_status() == 0
    return got


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (7, 2048, 6144), (64, 4096, 14336), (333, 768, 4096),
                                   (257, 1000, 1056)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantised_operands(m, n, k, dtype):
    """What the quantiser makes of normal values, with a bias of each type."""
    a, sa = mxfp4.quant_mxfp4(rand((m, k), 1))
    b, sb = mxfp4.quant_mxfp4(rand((n, k), 2, 0.02))
    va, vb = mxfp4.dequant_mxfp4(a, sa, torch.float32).double(), mxfp4.dequant_mxfp4(b, sb, torch.float32).double()
    near(a, sa, va, b, sb, vb, dtype)
    near(a, sa, va, b, sb, vb, dtype, rand((n,), 3, 0.1, dtype))


@pytest.mark.parametrize("m,n,k", [(3, 130, 320), (9, 130, 320), (130, 70, 320), (300, 270, 320)])
def test_strides_pointers_and_out(m, n, k):
    """Rows of wider matrices, pointers that TMA cannot take (copied), an unaligned or
    strided out, whose other bytes stay as they were."""
    a, sa, va = operand(m, k, 1, spread=9)
    b, sb, vb = operand(n, k, 2, spread=9)
    wide_a = torch.zeros((m, k), dtype=torch.uint8, device="cuda")
    wide_b = torch.zeros((n, k + 16), dtype=torch.uint8, device="cuda")
    for off in (16, 3):
        wide_a[:, off:off + k // 2], wide_b[:, off:off + k // 2] = a, b
        near(wide_a[:, off:off + k // 2], sa, va, wide_b[:, off:off + k // 2], sb, vb, torch.bfloat16)
    flat = torch.zeros(sa.numel() + 5, dtype=torch.uint8, device="cuda")
    flat[5:] = sa.reshape(-1)
    near(a, flat[5:].view(sa.shape), va, b, sb, vb, torch.bfloat16)
    for dtype in (torch.bfloat16, torch.float32):
        for off, width in ((1, n + 3), (8, n + 22), (0, n)):
            buf = torch.full((m, width), 7.0, dtype=dtype, device="cuda")
            out = buf[:, off:off + n]
            assert near(a, sa, va, b, sb, vb, dtype, out=out) is out
            out.fill_(7.0)
            assert buf.eq(7.0).all()


@pytest.mark.parametrize("n", [1, 255, 449, 1002, 4099])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_pair_tiles_of_any_width(n, dtype):
    """Widths that TMA cannot store, with a bias, into rows of an odd distance: the columns of a
    product with more weight rows, and nothing beside them."""
    m, k, rows = 700, 320, -(-n // 128) * 128
    a, sa = mxfp4.quant_mxfp4(rand((m, k), 1))
    w, sw = mxfp4.quant_mxfp4(rand((rows, k), 2))
    bias = rand((rows,), 3, 1.0, dtype)
    pair = Config(128, 256, split=4)
    want = mxfp4.w4a4_mm(a, w.t(), sa, sw, dtype, bias, config=pair)[:, :n]
    assert torch.equal(mxfp4.w4a4_mm(a, w[:n].t(), sa, sw, dtype, bias[:n], config=pair), want)
    buf = torch.full((m, n + 4 + n % 2), 7.0, dtype=dtype, device="cuda")
    out = mxfp4.w4a4_mm(a, w[:n].t(), sa, sw, dtype, bias[:n], config=pair, out=buf[:, 3:3 + n])
    assert torch.equal(out, want)
    out.fill_(7.0)
    assert buf.eq(7.0).all()


def test_nan_blocks_reach_their_rows_and_columns_only():
    a, sa = mxfp4.quant_mxfp4(rand((40, 512), 1))
    x = rand((40, 512), 1)
    x[7, 100] = float("inf")
    w = rand((200, 512), 2)
    w[150, 511] = float("nan")
    a, sa = mxfp4.quant_mxfp4(x)
    b, sb = mxfp4.quant_mxfp4(w)
    got = mxfp4.w4a4_mm(a, b.t(), sa, sb)
    pair = mxfp4.w4a4_mm(a, b.t(), sa, sb, config=Config(128, 256, split=4))
    assert torch.equal(got.isnan(), pair.isnan())
    few = mxfp4.w4a4_mm(a[5:9], b.t(), mxfp4.quant_mxfp4(x[5:9])[1], sb, config=Config(4, 0, split=5))
    assert torch.equal(few.isnan(), got[5:9].isnan())
    want = torch.zeros((40, 200), dtype=torch.bool, device="cuda")
    want[7], want[:, 150] = True, True
    assert torch.equal(got.isnan(), want) and torch.isfinite(got[~want]).all()


def test_scales_of_all_sizes():
    """Blocks from 2^-127 up: sums of very small and very large products."""
    for m in (4, 20, 150):
        a, sa, va = operand(m, 256, 5, spread=60)
        b, sb, vb = operand(140, 256, 6, spread=60)
        near(a, sa, va, b, sb, vb, torch.float32)
    lo = torch.zeros_like(sa)                     # every scale 2^-127: the products underflow
    got = mxfp4.w4a4_mm(a, b.t(), lo, sb, torch.float32)
    assert torch.isfinite(got).all()


def test_runs_repeat_bit_for_bit_and_graphs_replay():
    a, sa, _ = operand(50, 4096, 1, spread=20)
    b, sb, _ = operand(512, 4096, 2, spread=20)
    first = mxfp4.w4a4_mm(a, b.t(), sa, sb, torch.float32)
    for _ in range(5):
        assert torch.equal(mxfp4.w4a4_mm(a, b.t(), sa, sb, torch.float32), first)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mxfp4.w4a4_mm(a, b.t(), sa, sb, torch.float32))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s, g in zip(streams, graphs):            # both at once: the calls share nothing
        with torch.cuda.stream(s):
            for _ in range(20):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs)
    assert _native.read_status() == 0


def test_one_row_may_have_any_stride():
    a, sa, va = operand(1, 96, 1)
    b, sb, vb = operand(1, 96, 2)
    for cfg in (None, Config(1, 0, split=5), Config(16, 128, split=1), Config(128, 256, split=4)):
        for stride in (0, 5):
            x, w = torch.as_strided(a, (1, 48), (stride, 1)), torch.as_strided(b, (1, 48), (stride, 1))
            out = torch.as_strided(torch.empty(8, device="cuda"), (1, 1), (0, 1))
            got = mxfp4.w4a4_mm(x, w.t(), sa, sb, torch.float32, config=cfg, out=out)
            assert torch.equal(got.double(), va @ vb.t())


def test_weights_to_copy_are_refused_under_programmatic_launch():
    a, sa, va = operand(3, 64, 1)
    b, sb, vb = operand(40, 64, 2)
    odd = torch.zeros((40, 48), dtype=torch.uint8, device="cuda")
    odd[:, 3:35] = b
    int8_linear.set_pdl(True)
    try:
        with pytest.raises(NotSupported):
            mxfp4.w4a4_mm(a, odd[:, 3:35].t(), sa, sb)
        flat = torch.zeros(513, dtype=torch.uint8, device="cuda")
        flat[1:] = sb.reshape(-1)
        with pytest.raises(NotSupported):
            mxfp4.w4a4_mm(a, b.t(), sa, flat[1:].view(1, 1, 512))
        flat[1:] = sa.reshape(-1)
        mxfp4.w4a4_mm(a, b.t(), flat[1:].view(1, 1, 512), sb)       # an activation is copied
        mxfp4.w4a4_mm(a, b.t(), sa, torch.cat([sb, sb], 2)[:, :, :512])   # one tile: contiguous
        got = mxfp4.w4a4_mm(a, b.t(), torch.cat([sa, sa], 2)[:, :, :512], sb, torch.float32)
        assert torch.equal(got.double(), va @ vb.t())
    finally:
        int8_linear.set_pdl(False)


def test_refusals_and_empty():
    a, sa, _ = operand(4, 64, 1)
    b, sb, _ = operand(6, 64, 2)
    assert mxfp4.w4a4_mm(a[:0], b.t(), sa[:0], sb).shape == (0, 6)
    assert mxfp4.w4a4_mm(a, b[:0].t(), sa, sb[:0]).shape == (4, 0)
    for bad in ((a.to(torch.int8), b.t(), sa, sb), (a, b.t(), sa.to(torch.int8), sb), (a, b.t().contiguous(), sa, sb),
                (a[:, :24], b[:, :24].t(), sa, sb)):
        with pytest.raises(NotSupported):
            mxfp4.w4a4_mm(*bad)
    for bad in ((a, b[:, :16].t(), sa, sb), (a, b.t(), sa[:, :, :256], sb), (a, b.t(), sa, sb.cpu()),
                (a.cpu(), b.cpu().t(), sa.cpu(), sb.cpu())):
        with pytest.raises(ValueError):
            mxfp4.w4a4_mm(*bad)
    with pytest.raises(NotSupported):
        mxfp4.w4a4_mm(a, b.t(), sa, sb, torch.int8)
    with pytest.raises(NotSupported):
        mxfp4.w4a4_mm(a, b.t(), sa, sb, bias=torch.zeros(6, dtype=torch.int8, device="cuda"))
    with pytest.raises(ValueError):
        mxfp4.w4a4_mm(a, b.t(), sa, sb, bias=torch.zeros(5, device="cuda"))
    with pytest.raises(ValueError):
        mxfp4.w4a4_mm(a, b.t(), sa, sb, out=torch.zeros((4, 5), device="cuda"))
    for cfg in (Config(256, 128), Config(16, 0, split=5), Config(2, 0, split=5), Config(16, 128, split=3, cluster=2),
                Config(16, 128, split=1, stages=99)):
        with pytest.raises(NotSupported):
            mxfp4.w4a4_mm(a, b.t(), sa, sb, config=cfg)
    big, sbig, _ = operand(40, 64, 3)
    with pytest.raises(NotSupported):
        mxfp4.w4a4_mm(big, b.t(), sbig, sb, config=Config(16, 128, split=1))

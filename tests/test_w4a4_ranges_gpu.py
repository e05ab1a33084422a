"""The 4-bit product at both ends of the scale bytes, by value, on every kind of tile.

The factors' scales are extreme and their products are not: every block's sum is a normal
float32 number (or zero).  The bound is that of a float32 sum of K products in any order,
K * 2^-23 of the sum of their magnitudes, and half a step (2^-24) for the output."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int8_linear import Config, _native, mxfp4
from oracle import mxfp4 as om

pytestmark = pytest.mark.gpu

TILES = {"own choice": None, "CUDA cores": Config(4, 0, split=5), "split 16": Config(16, 128, swap_ab=True, split=1),
         "split 128, three CTAs": Config(128, 128, swap_ab=True, split=3, cluster=3),
         "pair": Config(128, 256, split=4)}


def operand(rows, k, low, high, seed):
    """Random codes with scale bytes low .. high: (q, s, float64 values)."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    tiles = om.tile_scales(torch.randint(low, high + 1, (rows, k // 32), generator=g, dtype=torch.uint8).numpy())
    return q.cuda(), torch.from_numpy(tiles).cuda(), om.operand_values(q.numpy(), tiles)


@pytest.mark.parametrize("tile", TILES)
@pytest.mark.parametrize("a_bytes,w_bytes", [((0, 0), (254, 254)), ((254, 254), (0, 0)), ((0, 8), (246, 254)),
                                             ((246, 254), (0, 8)), ((0, 240), (127, 127)), ((100, 100), (246, 246)),
                                             ((0, 0), (127, 254))])
def test_extreme_scales(tile, a_bytes, w_bytes):
    m, n, k = 4, 140, 1056
    a, sa, va = operand(m, k, *a_bytes, 1)
    w, sw, vw = operand(n, k, *w_bytes, 2)
    got = mxfp4.w4a4_mm(a, w.t(), sa, sw, torch.float32, config=TILES[tile]).double().cpu().numpy()
    want, size = va @ vw.T, np.abs(va) @ np.abs(vw).T
    assert size.max() < 2.0 ** 127 and size.min() > 2.0 ** -100
    assert (np.abs(got - want) <= size * (k * 2.0 ** -23) + np.abs(want) * 2.0 ** -24).all()
    assert _native.read_status() == 0


@pytest.mark.parametrize("tile", TILES)
def test_equal_fours(tile):
    """All codes 4 and one weight scale of 2^119: the sums leave float32's range only where the
    products do, and a NaN scale still makes its outputs NaN."""
    k = 1024
    four = torch.full((3, k // 2), 0x66, dtype=torch.uint8, device="cuda")
    for byte_a, byte_w in ((100, 246), (246, 100), (8, 254), (254, 8)):
        sa = torch.full((1, k // 128, 512), byte_a, dtype=torch.uint8, device="cuda")
        sw = torch.full((1, k // 128, 512), byte_w, dtype=torch.uint8, device="cuda")
        want = 16.0 * k * 2.0 ** (byte_a + byte_w - 254)
        got = mxfp4.w4a4_mm(four, four.t(), sa, sw, torch.float32, config=TILES[tile])
        assert got.eq(want).all(), (got, want)
        for s in (sa, sw):
            keep = s.clone()
            s[:] = 255
            assert mxfp4.w4a4_mm(four, four.t(), sa, sw, torch.float32, config=TILES[tile]).isnan().all()
            s.copy_(keep)

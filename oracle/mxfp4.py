"""MXFP4 in numpy: block quantisation, packing, the tiled scale layout, and the rows that
the fused quantisers make 4-bit values of (test infrastructure only).

Written from the definitions: a block of 32 values y has the scale 2^(floor(log2 max|y|) - 2),
at least 2^-127, and its values are y / scale rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3,
4, 6 (ties to the even code), saturated.  A block with an infinity or a NaN has scale byte
0xFF and zero codes."""

from __future__ import annotations

import numpy as np

from oracle.numerics import round_to

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
BLOCK = 32


def quantise(y: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes uint8 [R, K], scale bytes uint8 [R, K/32]) of float values y."""
    r, k = y.shape
    b = y.astype(np.float64).reshape(r, k // BLOCK, BLOCK)
    amax = np.abs(b).max(-1)
    bad = ~np.isfinite(b).all(-1)
    amax = np.where(bad, 1.0, amax)
    exp = np.where(amax > 0, np.frexp(amax)[1] - 1, -1000)     # floor(log2 amax)
    e = np.maximum(exp - 2, -127)
    with np.errstate(invalid="ignore"):
        mag = np.abs(np.where(bad[..., None], 0.0, b)) / np.exp2(e.astype(np.float64))[..., None]
    mid = (GRID[1:] + GRID[:-1]) / 2
    low, high = np.searchsorted(mid, mag, side="left"), np.searchsorted(mid, mag, side="right")
    code = np.where(low % 2 == 0, low, high)                  # differ only at a tie: the even one
    sign = np.signbit(np.where(bad[..., None], 0.0, b))
    codes = (code + 8 * sign).astype(np.uint8).reshape(r, k)
    return codes, np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes: np.ndarray) -> np.ndarray:
    return codes[:, 0::2] | (codes[:, 1::2] << 4)


def unpack(q: np.ndarray) -> np.ndarray:
    out = np.empty((q.shape[0], 2 * q.shape[1]), dtype=np.uint8)
    out[:, 0::2], out[:, 1::2] = q & 15, q >> 4
    return out


def tile_scales(s: np.ndarray) -> np.ndarray:
    """Scale bytes [R, blocks] in tiles [ceil(R/128), ceil(blocks/4), 512], zeros outside."""
    r, nb = s.shape
    out = np.zeros((-(-r // 128), -(-nb // 4), 512), dtype=np.uint8)
    for i in range(r):
        for j in range(nb):
            out[i // 128, j // 4, (i % 32) * 16 + (i // 32) % 4 * 4 + j % 4] = s[i, j]
    return out


def untile_scales(t: np.ndarray, rows: int, blocks: int) -> np.ndarray:
    i, j = np.arange(rows)[:, None], np.arange(blocks)[None]
    return t[i // 128, j // 4, (i % 32) * 16 + (i // 32) % 4 * 4 + j % 4]


def values(codes: np.ndarray, s: np.ndarray) -> np.ndarray:
    """float64 values of codes [R, K] with scale bytes [R, K/32]."""
    v = np.where(codes >= 8, -1.0, 1.0) * GRID[codes & 7]
    scale = np.where(s == 255, np.nan, np.exp2(s.astype(np.float64) - 127))
    return v * np.repeat(scale, BLOCK, axis=1)


def operand_values(q: np.ndarray, tiles: np.ndarray) -> np.ndarray:
    """float64 values of a packed operand and its tiled scales."""
    rows, k = q.shape[0], 2 * q.shape[1]
    return values(unpack(q), untile_scales(tiles, rows, k // BLOCK))


def silu_rows(gate_up: np.ndarray, act: str) -> np.ndarray:
    """y of silu(gate) * up: exact, rounded to float32, then to the activation type."""
    k = gate_up.shape[1] // 2
    g, u = gate_up[:, :k].astype(np.float64), gate_up[:, k:].astype(np.float64)
    with np.errstate(all="ignore"):
        return round_to((g / (1 + np.exp(-g)) * u).astype(np.float32), act)


def norm_rows(x: np.ndarray, residual: np.ndarray | None, weight: np.ndarray, eps: float, act: str,
              wdt: str) -> tuple[np.ndarray, np.ndarray]:
    """(y, residual_out) of add + RMSNorm: the sum in float32, 1/sqrt(mean + eps) rounded
    once to float32, then the two products in float32, rounded to the weight's and the
    activation's type."""
    with np.errstate(all="ignore"):
        h = x.astype(np.float32) if residual is None else x.astype(np.float32) + residual.astype(np.float32)
        mean = (h.astype(np.float64) ** 2).sum(-1, keepdims=True) / h.shape[1]
        r = (1 / np.sqrt(mean + eps)).astype(np.float32)
        y = round_to(round_to(h * r, wdt) * weight.astype(np.float32), act)
        return y, round_to(h, act)

"""4-bit operators and the query/key norm on tensors of more than 2^31 (the flat kernels:
2^33, where a call takes two launches) values: the rows around each border are those of a
call on these rows alone."""

from __future__ import annotations

import pytest
import torch

from int8_linear import mxfp4
from int8_linear.qk_norm import qk_norm_rope
from tests.gpu_util import rand

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(autouse=True)
def freed():
    yield
    torch.cuda.empty_cache()


def filled(m, k, seed, dtype=torch.bfloat16):
    """A matrix whose rows differ: 1000003 values over and over."""
    base = rand((1000003,), seed, 2.0, dtype)
    x = torch.empty(m * k, dtype=dtype, device="cuda")
    whole = x.numel() // base.numel()
    x[:whole * base.numel()].view(whole, -1).copy_(base)
    x[whole * base.numel():] = base[:x.numel() - whole * base.numel()]
    return x.view(m, k)


def windows(m, k, most):
    """256-row windows (from a multiple of 128) around the rows where an offset in values passes
    a power of two, and the last rows."""
    at = [(1 << p) // k // 128 * 128 - 128 for p in range(30, most + 1)]
    return [(lo, min(lo + 256, m)) for lo in at if 0 <= lo < m] + [((m - 1) // 128 * 128, m)]


def same(q, s, part, lo, hi):
    return torch.equal(q[lo:hi], part[0]) and torch.equal(s[lo // 128:(hi + 127) // 128], part[1])


def test_quant_and_dequant():
    m, k = (1 << 21) + 136, 4096
    x = filled(m, k, 1)
    q, s = mxfp4.quant_mxfp4(x)
    for lo, hi in windows(m, k, 33):
        assert same(q, s, mxfp4.quant_mxfp4(x[lo:hi]), lo, hi), lo
    del x
    out = mxfp4.dequant_mxfp4(q, s)
    for lo, hi in windows(m, k, 33):
        assert torch.equal(out[lo:hi], mxfp4.dequant_mxfp4(q[lo:hi], s[lo // 128:(hi + 127) // 128])), lo


def test_silu():
    m, k = (1 << 19) + 300, 4096
    gu = filled(m, 2 * k, 2)
    q, s = mxfp4.silu_mul_quant_mxfp4(gu)
    for lo, hi in windows(m, 2 * k, 32) + windows(m, k, 31):
        assert same(q, s, mxfp4.silu_mul_quant_mxfp4(gu[lo:hi]), lo, hi), lo


@pytest.mark.parametrize("m,k", [((1 << 19) + 300, 4096), ((1 << 22) + 300, 544)])
def test_norm(m, k):
    x, r, w = filled(m, k, 3), filled(m, k, 4), rand((k,), 5, 0.1) + 1
    q, s, out = mxfp4.add_rmsnorm_quant_mxfp4(x, r, w, EPS)
    for lo, hi in windows(m, k, 31):
        part = mxfp4.add_rmsnorm_quant_mxfp4(x[lo:hi], r[lo:hi], w, EPS)
        assert same(q, s, part, lo, hi) and torch.equal(out[lo:hi], part[2]), lo


def test_qk_norm_rope():
    m, heads, kv, d = (1 << 18) + 37, 48, 8, 128
    qkv = filled(m, (heads + 2 * kv) * d, 6)
    wq, wk, cs = rand((d,), 1, 0.2) + 1, rand((d,), 2, 0.2) + 1, rand((999, d), 3, 1.0, torch.float32)
    pos = torch.arange(m, device="cuda") % 999
    q, k = qk_norm_rope(qkv, wq, wk, EPS, pos, cs, heads, kv)
    for lo, hi in windows(m, (heads + 2 * kv) * d, 31) + windows(m, heads * d, 30):
        part = qk_norm_rope(qkv[lo:hi], wq, wk, EPS, pos[lo:hi], cs, heads, kv)
        assert torch.equal(q[lo:hi], part[0]) and torch.equal(k[lo:hi], part[1]), lo


@pytest.mark.parametrize("n", [32768, 32761])
def test_product(n):
    """K = 64 and scales close to one another, so that float32 holds every sum exactly and all
    tiles give the same bits."""
    m, k = 70001, 64
    a, sa = mxfp4.quant_mxfp4(filled(m, k, 7))
    b, sb = mxfp4.quant_mxfp4(rand((n, k), 8, 2.0))
    out = mxfp4.w4a4_mm(a, b.t(), sa, sb)
    for lo, hi in windows(m, n, 31):
        part = mxfp4.w4a4_mm(a[lo:hi], b.t(), sa[lo // 128:(hi + 127) // 128], sb)
        assert torch.equal(out[lo:hi], part), lo
        few = mxfp4.w4a4_mm(a[lo:lo + 17], b.t(), sa[lo // 128:lo // 128 + 1], sb)
        assert torch.equal(out[lo:lo + 17], few), lo


def test_product_of_a_weight_past_four_gigabytes():
    """Values of one size, so that every partial sum is exact in float32."""
    m, n, k = 20, (1 << 17) + 200, 65536
    a, sa = mxfp4.quant_mxfp4(rand((m, k), 9).sign())
    w, sw = mxfp4.quant_mxfp4(filled(n, k, 10).sign_())
    out = mxfp4.w4a4_mm(a, w.t(), sa, sw, torch.float32)
    for lo, hi in windows(n, k // 2, 32):
        part = mxfp4.w4a4_mm(a, w[lo:hi].t(), sa, sw[lo // 128:(hi + 127) // 128], torch.float32)
        assert torch.equal(out[:, lo:hi], part) and part.abs().max() > 100, lo

"""The 4-bit (MXFP4) quantisers and dequantisation against the numpy oracle
(oracle/mxfp4.py): codes and scale bytes are compared bit for bit, padding bytes of the
scale tiles included."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int8_linear import NotSupported, mxfp4
from oracle import mxfp4 as om
from oracle.numerics import to_bits
from tests.gpu_util import bits, np_, rand

pytestmark = pytest.mark.gpu
EPS = 1e-6
DT = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}


def check(q, s, y):
    codes, e = om.quantise(y)
    assert q.dtype == s.dtype == torch.uint8
    assert np.array_equal(np_(s), om.tile_scales(e))
    assert np.array_equal(np_(q), om.pack(codes))


def spread(shape, seed, dtype):
    """Normal values over many binades, so that blocks have different scales."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp2(torch.randint(-9, 9, shape, generator=g).float())
    return x.to(dtype).cuda()


@pytest.mark.parametrize("m,k", [(1, 32), (1, 2048), (3, 96), (127, 160), (128, 128), (129, 4096), (300, 1056),
                                 (7, 14336), (1025, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quant(m, k, dtype):
    x = spread((m, k), m + k, dtype)
    check(*mxfp4.quant_mxfp4(x), np_(x))


def test_quant_of_unaligned_and_strided_rows():
    wide = spread((65, 1000), 5, torch.bfloat16)
    for lo, hi in ((0, 512), (8, 968), (3, 899), (1, 33)):
        x = wide[:, lo:hi]
        check(*mxfp4.quant_mxfp4(x), np_(x))
    x = wide[::2, 4:964]
    check(*mxfp4.quant_mxfp4(x), np_(x))


def test_one_row_may_have_any_stride():
    flat = spread((512,), 3, torch.bfloat16)
    w = torch.ones(256, dtype=torch.bfloat16, device="cuda")
    for stride in (0, 1, 7, 300):
        x = torch.as_strided(flat, (1, 256), (stride, 1))
        check(*mxfp4.quant_mxfp4(x), np_(x))
        check(*mxfp4.silu_mul_quant_mxfp4(x), om.silu_rows(np_(x), "bf16"))
        q, s, r = mxfp4.add_rmsnorm_quant_mxfp4(x, x, w, EPS)
        check(q, s, om.norm_rows(np_(x), np_(x), np_(w), EPS, "bf16", "bf16")[0])
        back = mxfp4.dequant_mxfp4(torch.as_strided(q, q.shape, (stride, 1)), s)
        assert torch.equal(back, mxfp4.dequant_mxfp4(q, s))
    with pytest.raises(ValueError):
        mxfp4.quant_mxfp4(flat[:256].expand(4, 256))       # rows on top of one another


@pytest.mark.parametrize("m,k", [(600, 2048), (2500, 64), (2369, 4096), (2368, 8192), (3000, 8224)])
@pytest.mark.parametrize("lo", [0, 8, 16, 3])
def test_large_batches(m, k, lo):
    """The forms that large batches take (a block per thread), 32-byte, 16-byte and unaligned
    rows, against the same rows in small batches."""
    wide, res = rand((m, 2 * k + 16), 7), rand((m, k + 16), 8)
    w = rand((k,), 9, 0.1) + 1.0
    x, r, gu = wide[:, lo:lo + k], res[:, lo:lo + k], wide[:, lo:lo + 2 * k]
    for fn in (lambda rows: mxfp4.quant_mxfp4(x[rows]), lambda rows: mxfp4.silu_mul_quant_mxfp4(gu[rows]),
               lambda rows: mxfp4.add_rmsnorm_quant_mxfp4(x[rows], r[rows], w, EPS),
               lambda rows: mxfp4.add_rmsnorm_quant_mxfp4(x[rows], None, w, EPS)):
        full = fn(slice(None))
        for begin, end in ((0, 128), (m // 128 * 128 - 128, m)):
            part = fn(slice(begin, end))
            assert torch.equal(full[0][begin:end], part[0])
            assert torch.equal(full[1][begin // 128:], part[1]) if end == m else torch.equal(full[1][:1], part[1])
            if len(full) == 3 and full[2] is not None:
                assert torch.equal(full[2][begin:end], part[2])
    y, _ = om.norm_rows(np_(x[-40:]), np_(r[-40:]), np_(w), EPS, "bf16", "bf16")
    codes, _ = om.quantise(y)
    assert np.array_equal(np_(mxfp4.add_rmsnorm_quant_mxfp4(x, r, w, EPS)[0][-40:]), om.pack(codes))


def test_rounding_borders_and_signs():
    """Every border between two steps, the values just beside it and their negatives, at
    scales across the range; the block's largest value fixes the scale at 4 to 8 steps."""
    mids = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)
    v = np.concatenate([mids, np.nextafter(mids, np.float32(0)), np.nextafter(mids, np.float32(9)), om.GRID])
    rows = []
    for top in (4.0, 6.0, 7.99):
        for e in (-126, -60, -3, 0, 7, 100):
            row = np.concatenate([v, -v, [top, -0.0, 0.0, -top, 1e-30, -1e-30]]).astype(np.float32)
            row = np.concatenate([row, np.full((-len(row)) % 32, top, np.float32)])
            row[31::32] = top
            with np.errstate(under="ignore"):
                rows.append(np.ldexp(row, e).astype(np.float32))
    x = np.stack(rows)
    check(*mxfp4.quant_mxfp4(torch.from_numpy(x).cuda()), x)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_extreme_blocks(dtype):
    info = torch.finfo(dtype)
    x = torch.zeros((9, 64), dtype=dtype)
    x[1, 5] = info.max
    x[2, 40] = -info.max
    x[3, :] = info.tiny
    x[4, 3] = info.smallest_normal / 4       # subnormal
    x[5, 0], x[5, 33] = float("inf"), 1.0
    x[6, 63], x[6, 1] = float("nan"), 2.0
    x[7, 2] = -float("inf")
    x[8] = 1.0
    q, s = mxfp4.quant_mxfp4(x.cuda())
    check(q, s, x.float().numpy())
    back = np_(mxfp4.dequant_mxfp4(q, s, torch.float32))
    assert np.isnan(back[5, :32]).all() and np.isfinite(back[5, 32:]).all()
    assert np.isnan(back[6, 32:]).all() and np.isfinite(back[6, :32]).all()
    assert not back[0].any()


@pytest.mark.parametrize("m,k", [(1, 32), (129, 160), (300, 2048)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_dequant_of_any_codes_and_scales(m, k, dtype):
    """All codes, all scale bytes (0xFF for NaN among them), strided and odd pointers."""
    g = torch.Generator().manual_seed(m)
    q = torch.randint(0, 256, (m, k // 2), generator=g, dtype=torch.uint8)
    s = torch.randint(0, 256, (-(-m // 128), -(-k // 128), 512), generator=g, dtype=torch.uint8)
    want = om.operand_values(q.numpy(), s.numpy())
    with np.errstate(all="ignore"):
        want = to_bits(want.astype(np.float32), DT[dtype])
    wide = torch.zeros((m, k // 2 + 12), dtype=torch.uint8, device="cuda")
    flat = torch.empty(m * k // 2 + 1, dtype=torch.uint8, device="cuda")
    wide[:, 4:4 + k // 2], flat[1:] = q.cuda(), q.cuda().reshape(-1)
    for qq in (q.cuda(), wide[:, 4:4 + k // 2], flat[1:].view(m, -1)):
        got = mxfp4.dequant_mxfp4(qq, s.cuda(), dtype)
        nan = np.isnan(np_(got))
        assert np.array_equal(nan, np.isnan(om.operand_values(q.numpy(), s.numpy())))
        assert np.array_equal(bits(got)[~nan], want[~nan])


@pytest.mark.parametrize("m,k", [(1, 32), (1, 2048), (5, 96), (129, 1056), (64, 4096), (300, 2048), (2, 14336),
                                 (2, 32768)])
@pytest.mark.parametrize("has_res", [False, True])
def test_add_rmsnorm_quant(m, k, has_res):
    x = rand((m, k), m)
    r = rand((m, k), m + 1, 2.0) if has_res else None
    w = rand((k,), 99, 0.1) + 1.0
    q, s, rout = mxfp4.add_rmsnorm_quant_mxfp4(x, r, w, EPS)
    y, r0 = om.norm_rows(np_(x), np_(r) if has_res else None, np_(w), EPS, "bf16", "bf16")
    check(q, s, y)
    assert (rout is None) == (not has_res)
    if has_res:
        assert np.array_equal(bits(rout), to_bits(r0, "bf16"))


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("wdt", [torch.bfloat16, torch.float16, torch.float32])
def test_add_rmsnorm_quant_types_and_strides(act, wdt):
    m, k = 33, 544
    w = (rand((k + 1,), 3, 0.1, torch.float32) + 1.0).to(wdt)
    x, r = rand((m, k + 8), 1, dtype=act), rand((m, k + 8), 2, dtype=act)
    for lo in (0, 8, 3):
        for wv in (w[:k], w[1:]):
            xs, rs = x[:, lo:lo + k] if lo + k <= k + 8 else x[:, :k], r[:, lo:lo + k]
            q, s, rout = mxfp4.add_rmsnorm_quant_mxfp4(xs, rs, wv, EPS)
            y, r0 = om.norm_rows(np_(xs), np_(rs), np_(wv), EPS, DT[act], DT[wdt])
            check(q, s, y)
            assert np.array_equal(np_(rout), r0)


def test_norm_of_special_rows():
    """Zero rows, rows whose squares leave float32's range, and rows with inf or NaN (which
    come out as NaN blocks).  Row 3 is all NaN too: linspace's step leaves float32's range."""
    x = torch.zeros((7, 256), dtype=torch.bfloat16)
    x[1] = 1e30
    x[2] = 1e-30
    x[3] = torch.linspace(-2e38, 2e38, 256)
    x[4, 7] = float("nan")
    x[5, 200] = float("inf")
    x[6] = 1e38 * torch.linspace(-3, 3, 256)
    w = torch.ones(256, dtype=torch.bfloat16)
    q, s, _ = mxfp4.add_rmsnorm_quant_mxfp4(x.cuda(), None, w.cuda(), EPS)
    y, _ = om.norm_rows(x.float().numpy(), None, w.float().numpy(), EPS, "bf16", "bf16")
    check(q, s, y)
    back = np_(mxfp4.dequant_mxfp4(q, s, torch.float32))
    assert np.isfinite(back[:3]).all() and np.isnan(back[3]).all() and np.isfinite(back[6]).all()
    assert np.isnan(back[4]).all() and np.isnan(back[5]).any()


@pytest.mark.parametrize("eps", [1e-6, 0.0])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(40, 2048), (1900, 1024), (1200, 4096), (300, 8192)])
def test_norm_of_special_rows_among_others(m, k, act, eps):
    """Zeros, infinities, NaN, values whose squares leave float32's range and values below its
    normal range, in rows by themselves and beside ordinary ones, in small and large batches.
    Without eps the factor of a row of zeros or of the smallest values is infinite."""
    x, r = rand((m, k), 1, dtype=act), rand((m, k), 2, dtype=act)
    big, small, least = (3e38, 1e-30, 1e-39) if act == torch.bfloat16 else (65504.0, 1e-5, 6e-8)
    fills = [0.0, -0.0, big, -small, least, float("inf"), float("nan")]
    for i, v in enumerate(fills):
        x[i::17], r[i::17] = v, 0.0  # whole rows
        x[i + 7::17, i * 31 % k] = v  # one value
    x[14::17, ::3], r[14::17] = 0.0, 0.0
    x[15::17], r[15::17] = small, -small  # a sum of zero
    w = rand((k,), 3, 0.1, act) + 1.0
    for res in (None, r):
        q, s, rout = mxfp4.add_rmsnorm_quant_mxfp4(x, res, w, eps)
        y, r0 = om.norm_rows(np_(x), None if res is None else np_(r), np_(w), eps, DT[act], DT[act])
        check(q, s, y)
        if res is not None:
            assert np.array_equal(np_(rout), r0, equal_nan=True)


@pytest.mark.parametrize("m,k", [(1, 32), (1, 6144), (33, 1056), (8, 14336), (300, 6144)])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_silu_mul_quant(m, k, act):
    gu = rand((m, 2 * k), m, 2.0, dtype=act)
    check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), DT[act]))


def test_silu_of_strided_rows():
    wide = rand((17, 1000), 4, 2.0)
    for lo, hi in ((0, 960), (3, 899), (8, 72)):
        gu = wide[:, lo:hi]
        check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), "bf16"))


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_silu_of_all_gates(act):
    """Every finite 16-bit gate, infinities and NaN, against ups of several sizes: overflow
    of exp, results below float32's normal range, exact zeros."""
    gates = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(act).view(-1, 32)
    for up in (1.0, -0.0, 3.0e-5, 1.5, 57344.0):
        ups = torch.full_like(gates, up)
        ups[:, 1::2] *= 0.75
        gu = torch.cat([gates, ups], 1).cuda()
        check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), DT[act]))


@pytest.mark.parametrize("lo", [0, 16, 8, 1])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_silu_of_large_batches(act, lo):
    """Enough blocks for the kernel with a thread per block, at each alignment of its loads."""
    gu = rand((401, 2 * 6144 + 32), 3, 2.0, dtype=act)[:, lo:lo + 2 * 6144]
    check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), DT[act]))


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_silu_of_all_gates_in_a_large_batch(act):
    """Every 16-bit gate in the kernel with a thread per block, against ups from zero over the
    smallest to the largest: blocks of zeros, blocks whose values all lie below float32's
    normal range, and such values beside normal ones."""
    gates = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(act).view(-1, 32)
    top = 126 if act == torch.bfloat16 else 15
    ups = [0.0, -0.0, *(1.3125 * 2.0**e * (-1) ** e for e in torch.linspace(-top, top, 36).round().int().tolist())]
    rows = []
    for i, up in enumerate(ups):
        u = torch.full(gates.shape, up, dtype=torch.float64)
        if i % 3 == 0:
            u[:, 1::2] *= 2.0**-20
        rows.append(torch.cat([gates, u.to(act)], 1))
    gu = torch.cat(rows).cuda()
    assert gu.shape[0] >= 512 * torch.cuda.get_device_properties(0).multi_processor_count
    check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), DT[act]))


@pytest.mark.parametrize("rows", [20, 410])
def test_silu_of_deep_gates_beside_ordinary_ones(rows):
    """bf16 gates so negative that 1 / (1 + exp(-gate)) leaves float32's normal range, with ups
    so large that the product does not, beside ordinary values of the product's size."""
    g = torch.Generator().manual_seed(rows)
    gate = -80.0 - 30.0 * torch.rand((rows, 6144), generator=g, dtype=torch.float64)
    up = 10.0 ** (36.0 + 2.5 * torch.rand((rows, 6144), generator=g, dtype=torch.float64))
    up *= torch.randint(0, 2, up.shape, generator=g) * 2 - 1
    size = (gate * torch.exp(gate) * up).abs()
    plain = torch.rand((rows, 6144), generator=g) < 0.5
    near = size.view(rows, -1, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(rows, -1)
    near = near * torch.exp2(-8.0 * torch.rand((rows, 1), generator=g, dtype=torch.float64))
    up = torch.where(plain, near * torch.randn(up.shape, generator=g), up)
    gate = torch.where(plain, torch.randn(up.shape, generator=g).double(), gate)
    gate[:, 5::640] = -1e30
    gu = torch.cat([gate, up], 1).to(torch.bfloat16).cuda()
    check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), "bf16"))


@pytest.mark.parametrize("rows", [20, 410])
@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
def test_silu_of_padded_batches(act, rows):
    """Rows of zeros, of zero gates and of zero ups, by turns with others."""
    gu = rand((rows, 2 * 6144), 5, 2.0, dtype=act)
    gu[1::4] = 0.0
    gu[2::4, :6144] = -0.0
    gu[3::4, 6144:] = 0.0
    check(*mxfp4.silu_mul_quant_mxfp4(gu), om.silu_rows(np_(gu), DT[act]))


def test_empty_batches():
    for k in (0, 64):
        q, s = mxfp4.quant_mxfp4(torch.empty((0, k), dtype=torch.bfloat16, device="cuda"))
        assert q.shape == (0, k // 2) and s.shape == (0, -(-k // 128), 512)
        assert mxfp4.dequant_mxfp4(q, s).shape == (0, k)
        q, s = mxfp4.silu_mul_quant_mxfp4(torch.empty((0, 2 * k), dtype=torch.bfloat16, device="cuda"))
        assert q.shape == (0, k // 2)
    q, s = mxfp4.quant_mxfp4(torch.empty((5, 0), dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (5, 0) and mxfp4.dequant_mxfp4(q, s).shape == (5, 0)


def test_refusals():
    x = rand((4, 64), 1)
    w = rand((64,), 2)
    q, s = mxfp4.quant_mxfp4(x)
    with pytest.raises(NotSupported):
        mxfp4.quant_mxfp4(x[:, :48])
    with pytest.raises(NotSupported):
        mxfp4.quant_mxfp4(x.t())
    with pytest.raises(NotSupported):
        mxfp4.quant_mxfp4(x.to(torch.float64))
    with pytest.raises(NotSupported):
        mxfp4.silu_mul_quant_mxfp4(x.float())
    with pytest.raises(ValueError):
        mxfp4.add_rmsnorm_quant_mxfp4(x, x[:2], w, EPS)
    with pytest.raises(ValueError):
        mxfp4.add_rmsnorm_quant_mxfp4(x, None, w[:32], EPS)
    with pytest.raises(ValueError):
        mxfp4.add_rmsnorm_quant_mxfp4(x, None, w.cpu(), EPS)
    with pytest.raises(ValueError):
        mxfp4.dequant_mxfp4(q, s[:, :, :256])
    with pytest.raises(ValueError):
        mxfp4.dequant_mxfp4(q, s.cpu())
    with pytest.raises(NotSupported):
        mxfp4.dequant_mxfp4(q, s, torch.int8)
    with pytest.raises(NotSupported):
        mxfp4.add_rmsnorm_quant_mxfp4(rand((1, 65536), 1), None, rand((65536,), 2), EPS)


def test_custom_ops_opcheck():
    x, r, w = rand((9, 256), 1), rand((9, 256), 2), rand((256,), 3) + 1.0
    torch.library.opcheck(mxfp4.quant_mxfp4_op, (x,))
    torch.library.opcheck(mxfp4.rmsnorm_quant_mxfp4_op, (x, w, EPS))
    torch.library.opcheck(mxfp4.add_rmsnorm_quant_mxfp4_op, (x, r, w, EPS))
    torch.library.opcheck(mxfp4.silu_mul_quant_mxfp4_op, (x,))
    a, sa = mxfp4.quant_mxfp4(x)
    b, sb = mxfp4.quant_mxfp4(r)
    torch.library.opcheck(mxfp4.w4a4_mm_op, (a, b.t(), sa, sb, torch.bfloat16, None))


def test_two_streams_and_graph_replay():
    """Each call runs on the caller's stream; a captured call reads its inputs again at
    every replay."""
    x = spread((130, 512), 1, torch.bfloat16)
    want = mxfp4.quant_mxfp4(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mxfp4.quant_mxfp4(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = mxfp4.quant_mxfp4(x)
    other = spread((130, 512), 2, torch.bfloat16)
    x.copy_(other)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, mxfp4.quant_mxfp4(other)))

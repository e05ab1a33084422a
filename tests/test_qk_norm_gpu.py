"""qk_norm_rope against a float64 restatement.

Tolerance: the output's own rounding, half a step of its type (finfo.eps / 2 relative, half
the smallest subnormal absolute), and the float32 arithmetic before it.  There, a sum of D
squares is off by at most D 2^-24 relative in any order, its root by half of that, and the
mean, the root, the reciprocal and the products with x, the weight and the angle add at most
8 roundings: (D/2 + 8) 2^-24 of each of the two terms of a rotated value, and one more
rounding for their sum.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int8_linear import NotSupported
from int8_linear.qk_norm import qk_norm_rope, qk_norm_rope_op
from tests.gpu_util import np_, rand

pytestmark = pytest.mark.gpu
EPS = 1e-6


def table(length, rot, dtype=torch.float32, base=1e4):
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))
    angle = torch.arange(length, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).to(dtype).cuda()


def oracle(x, w, eps, cos, sin, rot, interleaved):
    """(y, bound) of heads x [M, H, D] in float64."""
    d = x.shape[2]
    n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    first = np.arange(rot // 2) * (2 if interleaved else 1)
    second = first + (1 if interleaved else rot // 2)
    y, size = n.copy(), np.abs(n)
    a, b = n[..., first], n[..., second]
    y[..., first], size[..., first] = a * cos - b * sin, np.abs(a * cos) + np.abs(b * sin)
    y[..., second], size[..., second] = b * cos + a * sin, np.abs(b * cos) + np.abs(a * sin)
    return y, size * (d / 2 + 9) * 2.0 ** -24


def check(qkv, wq, wk, pos, cs, heads, kv, interleaved, got):
    d, rot, m = wq.numel(), cs.shape[1], qkv.shape[0]
    x = np_(qkv)[:, :(heads + kv) * d].astype(np.float64).reshape(m, heads + kv, d)
    t = np_(cs).astype(np.float64)[np_(pos)]
    cos, sin = t[:, None, :rot // 2], t[:, None, rot // 2:]
    info = torch.finfo(qkv.dtype)
    for out, part, w in ((got[0], x[:, :heads], wq), (got[1], x[:, heads:], wk)):
        y, bound = oracle(part, np_(w).astype(np.float64), EPS, cos, sin, rot, interleaved)
        tol = bound + (np.abs(y) + bound) * info.eps / 2 + info.tiny * info.eps / 2
        assert out.dtype == qkv.dtype and tuple(out.shape) == y.shape
        err = np.abs(np_(out).astype(np.float64) - y)
        assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("m,heads,kv,d,rot,interleaved", [
    (1, 16, 8, 128, 128, False), (1, 32, 8, 128, 128, True), (3, 4, 1, 64, 64, False), (17, 2, 2, 96, 96, False),
    (5, 3, 1, 80, 32, False), (9, 8, 2, 256, 64, True), (130, 5, 3, 256, 256, False), (1000, 16, 8, 128, 64, False),
    (7, 1, 0, 8, 8, True), (7, 0, 3, 16, 16, False), (2, 6, 2, 24, 16, True), (4, 7, 1, 128, 0, False),
    (4097, 12, 4, 128, 128, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_against_float64(m, heads, kv, d, rot, interleaved, dtype):
    qkv = rand((m, (heads + 2 * kv) * d), m + d, 3.0, dtype)
    wq, wk = rand((d,), 1, 0.2, dtype) + 1, rand((d,), 2, 0.2, dtype) + 1
    g = torch.Generator().manual_seed(m)
    pos = torch.randint(0, 999, (m,), generator=g).cuda()
    pos[0] = 998
    cs = table(999, rot)
    keep = qkv.clone()
    for p in (pos, pos.int()):
        check(qkv, wq, wk, p, cs, heads, kv, interleaved,
              qk_norm_rope(qkv, wq, wk, EPS, p, cs, heads, kv, interleaved=interleaved))
    assert torch.equal(qkv, keep)


@pytest.mark.parametrize("m,heads,kv,d,rot,interleaved", [
    (3000, 5, 2, 128, 128, False), (2003, 3, 4, 256, 64, True), (10007, 7, 1, 32, 16, False), (26001, 3, 0, 24, 24, True),
    (160001, 1, 0, 8, 8, True), (40000, 0, 1, 64, 32, False)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_batches(m, heads, kv, d, rot, interleaved, dtype):
    """CTAs that take several groups of heads: odd numbers of heads, a group with a query and a
    key head, results in place, tokens without angles and heads that are zero, infinite or NaN
    among others."""
    qkv = rand((m, (heads + 2 * kv) * d), d, 3.0, dtype)
    wq, wk = rand((d,), 1, 0.2, dtype) + 1, rand((d,), 2, 0.2, dtype) + 1
    pos = torch.randint(0, 999, (m,), generator=torch.Generator().manual_seed(m)).cuda()
    cs = table(999, rot)
    want = qk_norm_rope(qkv, wq, wk, EPS, pos, cs, heads, kv, interleaved=interleaved)
    check(qkv, wq, wk, pos, cs, heads, kv, interleaved, want)
    # Rows do not depend on the batch: a slice by itself takes the small batches' kernel.
    for lo in (0, m // 2, m - 5):
        part = qk_norm_rope(qkv[lo:lo + 5].contiguous(), wq, wk, EPS, pos[lo:lo + 5], cs, heads, kv,
                            interleaved=interleaved)
        assert all(torch.equal(a[lo:lo + 5], b) for a, b in zip(want, part))
    work = qkv.clone()
    got = qk_norm_rope(work, wq, wk, EPS, pos, cs, heads, kv, interleaved=interleaved,
                       q_out=work[:, :heads * d].view(m, heads, d),
                       k_out=work[:, heads * d:(heads + kv) * d].view(m, kv, d))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(work[:, (heads + kv) * d:], qkv[:, (heads + kv) * d:])

    pos[3::7] = torch.tensor([-1, 999, 2 ** 40], device="cuda").repeat(m)[:pos[3::7].numel()]
    qkv[1::5, :d], qkv[2::5, d // 2], qkv[4::5, d - 1] = 0.0, float("inf"), float("nan")
    got = qk_norm_rope(qkv, wq, wk, EPS, pos, cs, heads, kv, interleaved=interleaved)
    spoilt = torch.zeros(m, heads + kv, dtype=torch.bool, device="cuda")
    spoilt[2::5, 0] = spoilt[4::5, 0] = True
    spoilt[3::7] = True
    zero = torch.zeros_like(spoilt)
    zero[1::5, 0] = True
    out, was = torch.cat(got, 1), torch.cat(want, 1)
    assert torch.equal(out.isfinite().all(-1), ~spoilt)
    assert out[zero & ~spoilt].eq(0).all()
    fine = ~spoilt & ~zero
    assert torch.equal(out[fine], was[fine])


@pytest.mark.parametrize("wdt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tdt", [torch.bfloat16, torch.float16, torch.float32])
def test_weight_and_angle_types_and_odd_pointers(wdt, tdt):
    m, heads, kv, d, rot = 11, 4, 2, 128, 48
    qkv = rand((m, 1024), 3)
    w = rand((2 * d + 2,), 1, 0.2, torch.float32).to(wdt) + 1
    cs = table(64, rot, tdt)
    flat = torch.empty(cs.numel() + 1, dtype=tdt, device="cuda")
    flat[1:] = cs.reshape(-1)
    pos = torch.arange(m).cuda()
    for wq, wk in ((w[:d], w[d:2 * d]), (w[1:d + 1], w[d + 1:2 * d + 1])):
        for t in (cs, flat[1:].view(64, rot)):
            check(qkv, wq, wk, pos, t, heads, kv, False, qk_norm_rope(qkv, wq, wk, EPS, pos, t, heads, kv))


def test_in_place_and_into_wider_rows():
    """q_out and k_out may be the heads' own places in qkv (the values behind them stay as
    they were), or rows of a wider buffer."""
    m, heads, kv, d = 37, 6, 2, 64
    qkv = rand((m, (heads + 2 * kv) * d), 5)
    wq, wk = rand((d,), 1, 0.2) + 1, rand((d,), 2, 0.2) + 1
    cs, pos = table(100, d), torch.arange(m).cuda() * 2
    q, k = qk_norm_rope(qkv, wq, wk, EPS, pos, cs, heads, kv)
    work = qkv.clone()
    qv = work[:, :heads * d].view(m, heads, d)
    kview = work[:, heads * d:(heads + kv) * d].view(m, kv, d)
    got = qk_norm_rope(work, wq, wk, EPS, pos, cs, heads, kv, q_out=qv, k_out=kview)
    assert got[0] is qv and got[1] is kview
    assert torch.equal(qv, q) and torch.equal(kview, k)
    assert torch.equal(work[:, (heads + kv) * d:], qkv[:, (heads + kv) * d:])
    cache = torch.full((m + 2, 2, kv, d), 7.0, dtype=torch.bfloat16, device="cuda")
    qk_norm_rope(qkv, wq, wk, EPS, pos, cs, heads, kv, k_out=cache[1:m + 1, 0])
    assert torch.equal(cache[1:m + 1, 0], k)
    cache[1:m + 1, 0] = 7.0
    assert cache.eq(7.0).all()


def test_positions_outside_the_table_give_nan_and_no_others_do():
    qkv = rand((6, 3 * 64), 1)
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor([0, -1, 31, 32, 2 ** 40, 5], device="cuda")
    q, k = qk_norm_rope(qkv, w, w, EPS, pos, table(32, 32), 2, 1)
    bad = torch.tensor([False, True, False, True, True, False], device="cuda")
    assert torch.equal(q.isnan().all(-1).all(-1), bad) and torch.equal(q.isnan().any(-1).any(-1), bad)
    assert torch.equal(k.isnan().all(-1).all(-1), bad) and torch.equal(k.isnan().any(-1).any(-1), bad)
    q, _ = qk_norm_rope(qkv, w, w, EPS, pos, table(0, 0), 2, 1)      # no rotation: no angles needed
    assert torch.isfinite(q).all()


def test_one_token_may_have_any_stride_and_the_op_checks():
    flat, w, cs = rand((400,), 1), torch.ones(64, dtype=torch.bfloat16, device="cuda"), table(9, 64)
    pos = torch.tensor([4], device="cuda")
    want = qk_norm_rope(flat[:256].view(1, 256), w, w, EPS, pos, cs, 3, 1)
    for stride in (0, 3):
        got = qk_norm_rope(torch.as_strided(flat, (1, 256), (stride, 1)), w, w, EPS, pos, cs, 3, 1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.library.opcheck(qk_norm_rope_op, (flat[:256].view(1, 256), w, w, EPS, pos, cs, 3, 1, False))


def test_special_heads_keep_to_themselves():
    """A zero head stays zero; a head with an infinity or a NaN spoils no other."""
    qkv = rand((4, 4 * 64), 1)
    qkv[0, :64] = 0
    qkv[1, 70] = float("inf")
    qkv[2, 130] = float("nan")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    q, k = qk_norm_rope(qkv, w, w, EPS, torch.arange(4).cuda(), table(9, 64), 3, 1)
    assert q[0, 0].eq(0).all()
    fine = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    fine[1, 1] = fine[2, 2] = False
    assert torch.equal(torch.isfinite(q).all(-1), fine) and torch.isfinite(k).all()


def test_empty_refusals_and_streams():
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    cs = table(8, 64)
    pos = torch.zeros(3, dtype=torch.int64, device="cuda")
    qkv = rand((3, 256), 1)
    q, k = qk_norm_rope(qkv[:0], w, w, EPS, pos[:0], cs, 2, 1)
    assert q.shape == (0, 2, 64) and k.shape == (0, 1, 64)
    with pytest.raises(NotSupported):
        qk_norm_rope(qkv.float(), w, w, EPS, pos, cs, 2, 1)
    with pytest.raises(NotSupported):
        qk_norm_rope(qkv[:, 1:], w, w, EPS, pos, cs, 2, 1)
    with pytest.raises(NotSupported):
        qk_norm_rope(qkv, w, w, EPS, pos, cs[:, :8].contiguous(), 2, 1)
    with pytest.raises(NotSupported):
        qk_norm_rope(rand((3, 2048), 1), rand((512,), 1), rand((512,), 1), EPS, pos, cs, 2, 1)
    with pytest.raises(ValueError):
        qk_norm_rope(qkv, w, w, EPS, pos, cs, 4, 1)
    with pytest.raises(ValueError):
        qk_norm_rope(qkv, w, w.float(), EPS, pos, cs, 2, 1)
    with pytest.raises(ValueError):
        qk_norm_rope(qkv, w, w, EPS, pos.float(), cs, 2, 1)
    with pytest.raises(ValueError):
        qk_norm_rope(qkv, w, w, EPS, pos.cpu(), cs, 2, 1)
    with pytest.raises(ValueError):
        qk_norm_rope(qkv, w, w, EPS, pos, cs, 2, 1, q_out=qkv[:, :128])
    want = qk_norm_rope(qkv, w, w, EPS, pos, cs, 2, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = qk_norm_rope(qkv, w, w, EPS, pos, cs, 2, 1)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

"""qk_norm_rope on heads of all of bf16's range: a head's result does not depend on its size
where eps does not count, however large or small its squares are.

The bound is that of the other tests of this operator (see test_qk_norm_gpu)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from int8_linear.qk_norm import qk_norm_rope
from tests.gpu_util import np_, rand
from tests.test_qk_norm_gpu import oracle, table

pytestmark = pytest.mark.gpu


def heads_of_all_sizes(m, heads, d, seed):
    """Head h of token t has values of about 2^e with e from -130 to 125, some of them smaller
    by up to 2^40; every third head is plain."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-130, 126, (m, heads, 1), generator=g)
    e[:, ::3] = 0
    down = torch.randint(0, 41, (m, heads, d), generator=g) * (torch.rand((m, heads, d), generator=g) < 0.3)
    x = torch.rand((m, heads, d), generator=g, dtype=torch.float64) + 0.5
    x = x * torch.where(torch.rand((m, heads, d), generator=g) < 0.5, -1.0, 1.0) * torch.exp2((e - down).double())
    return x.to(torch.bfloat16).cuda()


@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e-35, 1e30])
@pytest.mark.parametrize("m,heads,kv,d,rot,interleaved", [(5, 6, 3, 128, 128, False), (40, 7, 1, 256, 64, True),
                                                          (64, 3, 2, 8, 8, True), (3000, 5, 2, 128, 64, False),
                                                          (9000, 4, 1, 24, 16, True)])
def test_heads_of_all_sizes(m, heads, kv, d, rot, interleaved, eps):
    x = heads_of_all_sizes(m, heads + kv, d, m)
    wq, wk = rand((d,), 1, 0.2) + 1, rand((d,), 2, 0.2) + 1
    pos = torch.randint(0, 99, (m,), generator=torch.Generator().manual_seed(1)).cuda()
    cs = table(99, rot)
    got = qk_norm_rope(x.view(m, -1), wq, wk, eps, pos, cs, heads, kv, interleaved=interleaved)
    t = np_(cs).astype(np.float64)[np_(pos)]
    cos, sin = t[:, None, :rot // 2], t[:, None, rot // 2:]
    values = np_(x).astype(np.float64)
    info = torch.finfo(torch.bfloat16)
    for out, part, w in ((got[0], values[:, :heads], wq), (got[1], values[:, heads:], wk)):
        y, bound = oracle(part, np_(w).astype(np.float64), np.float64(np.float32(eps)), cos, sin, rot, interleaved)
        assert np.isfinite(y).all()
        tol = bound + (np.abs(y) + bound) * info.eps / 2 + info.tiny * info.eps / 2
        err = np.abs(np_(out).astype(np.float64) - y)
        assert (err <= tol).all(), (err - tol).max()


@pytest.mark.parametrize("m", [4, 3000])
def test_plain_heads_beside_others_keep_their_bits(m):
    heads, d = 6, 128
    x = rand((m, heads * d), 3)
    w = rand((d,), 1, 0.2) + 1
    pos, cs = torch.arange(m).cuda() % 99, table(99, d)
    want, _ = qk_norm_rope(x, w, w, 1e-6, pos, cs, heads, 0)
    odd = x.clone().view(m, heads, d)
    odd[:, 1], odd[:, 2, 5], odd[:, 4, 7] = odd[:, 1] * 2.0 ** 100, float("nan"), float("inf")
    got, _ = qk_norm_rope(odd.view(m, -1), w, w, 1e-6, pos, cs, heads, 0)
    assert torch.equal(got[:, [0, 3, 5]], want[:, [0, 3, 5]])
    assert got[:, 2].isnan().all() and got[:, 1].isfinite().all() and got[:, 1].ne(0).any(-1).all()
    # x / sqrt(inf) is 0 for every finite x, and inf / inf NaN, which reaches the value it is rotated with
    nan = torch.zeros(d, dtype=torch.bool, device="cuda")
    nan[7], nan[7 + d // 2] = True, True
    assert got[:, 4][:, nan].isnan().all() and got[:, 4][:, ~nan].eq(0).all()


def test_one_token_may_have_any_distance():
    heads, kv, d = 3, 1, 24
    x, w = rand((1, (heads + kv) * d), 5), rand((d,), 1, 0.2) + 1
    pos, cs = torch.tensor([7]).cuda(), table(99, 16)
    want = qk_norm_rope(x, w, w, 1e-6, pos, cs, heads, kv)
    buf = torch.zeros(300, dtype=torch.bfloat16, device="cuda")
    for stride in (0, 5, 101):
        q, k = (torch.as_strided(buf, (1, n, d), (stride, d, 1), 96 * i) for i, n in ((1, heads), (2, kv)))
        row = torch.as_strided(buf, (1, (heads + kv) * d), (stride, 1))
        row.copy_(x)
        got = qk_norm_rope(row, w, w, 1e-6, pos, cs, heads, kv, q_out=q, k_out=k)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

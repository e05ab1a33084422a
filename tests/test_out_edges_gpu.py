"""w8a8_mm into `out` views inside wider rows: the bytes beside the view stay as they were,
also where a row of outputs does not end on a 16-byte boundary (a TMA store ends there, so
such rows take plain stores)."""

from __future__ import annotations

import pytest
import torch

from int8_linear import Config, w8a8_mm
from tests.gpu_util import ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cfg", [Config(128, 256), Config(128, 256, split=4), Config(256, 128), Config(64, 128, split=3, cluster=2),
                                 Config(64, 128, store=1), Config(128, 256, split=2)], ids=lambda c: c.name)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n", [270, 271, 264])
def test_bytes_beside_the_view_stay(cfg, dtype, n):
    m, k = 64 if cfg.bm == 64 else 300, 320
    a, w, one = ints((m, k), 1), ints((n, k), 2), torch.ones(1, device="cuda")
    want = w8a8_mm(a, w.t(), one, one, dtype, config=cfg)
    for off, width in ((8, 288), (0, 296), (1, 280)):
        buf = torch.full((m, width), 7.0, dtype=dtype, device="cuda")
        out = buf[:, off:off + n]
        w8a8_mm(a, w.t(), one, one, dtype, config=cfg, out=out)
        assert torch.equal(out, want)
        out.fill_(7.0)
        assert buf.eq(7.0).all()

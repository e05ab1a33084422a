"""First calls of two host threads at once, which want different amounts of shared memory of
the same kernel: both succeed, and so does every later call.  Each attempt is a process of its
own, as a kernel's first call in a process is the one that matters."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import threading
import torch
from int8_linear import Config, mxfp4, w8a8_mm

k = 4096
a, sa = mxfp4.quant_mxfp4(torch.randn(16, k, device="cuda"))
w, sw = mxfp4.quant_mxfp4(torch.randn(256, k, device="cuda"))
x = torch.ones(16, k, dtype=torch.int8, device="cuda")
y = torch.ones(256, k, dtype=torch.int8, device="cuda")
one = torch.ones(1, device="cuda")

def four(bm, bn, split, stages, dtype=torch.bfloat16):
    mxfp4.w4a4_mm(a, w.t(), sa, sw, dtype, config=Config(bm, bn, swap_ab=None if split == 4 else True, split=split, stages=stages))

def eight(bm, bn, stages, m=16, split=1):
    w8a8_mm(x[:m], y.t(), one, one, config=Config(bm, bn, stages=stages, split=split))

calls = [lambda s, t=t: four(t, 128, 1, s + 1) for t in (16, 32, 64, 128)]
calls += [lambda s, d=d: four(128, 256, 4, s + 2, d) for d in (torch.bfloat16, torch.float16, torch.float32)]
calls += [lambda s, t=t: eight(t, 128, s + 2) for t in (16, 32, 64)]
calls += [lambda s, t=t: eight(128, t, s + 2) for t in (128, 256)]
calls += [lambda s, t=t: eight(t, 0, 1 + s, min(t, 16), 5) for t in (1, 2, 4, 8)]
torch.cuda.synchronize()
errors = []
for call in calls:
    barrier = threading.Barrier(2)

    def run(more):
        barrier.wait()
        try:
            call(more)
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(more,)) for more in (0, 2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for more in (0, 2, 1):
        try:
            call(more)
        except Exception as e:
            errors.append(e)
torch.cuda.synchronize()
assert not errors, errors
"""


@pytest.mark.parametrize("attempt", range(4))
def test_first_calls_of_two_threads(attempt):
    done = subprocess.run([sys.executable, "-c", CODE], cwd=Path(__file__).resolve().parent.parent, timeout=300,
                          capture_output=True, text=True)
    assert done.returncode == 0, done.stderr[-2000:]

"""Block operators at widths, views, sizes and values that the calls accept and that are easily got wrong, against their
formulas in 64 bits (bounds and helpers as in test_gpu_block_ops)."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_block_ops import BF16, F16, block64, gen, near, ops, rand  # noqa: F401  (ops: fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant,t,rms", [(False, BF16, False), (False, F16, True), (True, BF16, True)])
@pytest.mark.parametrize("C", [1288, 1408, 1536, 1544, 1792, 2040])
@pytest.mark.parametrize("rows", [1, 5000])
def test_block_norm_six_and_seven_warps(ops, rows, C, quant, t, rms):
    g = gen(rows + C)
    h, r = rand(g, rows, C, at=0.3, t=t), rand(g, rows, C, by=3.0, t=t)
    post, pre = (rand(g, C, by=0.2, at=1.0), None if rms else rand(g, C)), (rand(g, C, by=0.2, at=1.0), None if rms else rand(g, C))
    gate = rand(g, C)
    x, y = ops.block_norm(h, r, post=post, pre=pre, gate=gate, res_scale=0.75, rms=rms)
    x64, ex, y64, ey = block64(h, r, post, pre, gate, 0.75, rms)
    near(x, x64, ex)
    near(y, y64, ey)
    if quant:
        x2, yq, s = ops.block_norm_quant_i8(h, r, post, pre, gate=gate, res_scale=0.75, rms=rms)
        q2, s2 = ops.quant_rows_i8(y)
        assert torch.equal(x2, x) and torch.equal(s, s2) and torch.equal(yq, q2)


@pytest.mark.parametrize("rows", [1, 5000])
def test_block_norm_six_warps_first_in_a_process(rows):
    """Each kernel's shared-memory limit belongs to the process: six warps may not live on what wider calls left behind."""
    code = f"""
import torch
from segment_anything_fast_b200 import ops
for t in (torch.bfloat16, torch.float16):
    for rms in (False, True):
        for C in (1536, 1288, 1792):
            h = torch.ones({rows}, C, dtype=t, device="cuda")
            f = torch.ones(C, device="cuda")
            x, y = ops.block_norm(h, h, pre=(f, None), rms=rms)
            assert (x == 2).all() and (y == (1 if rms else 0)).all()
            if t is torch.bfloat16:
                x, q, s = ops.block_norm_quant_i8(h, h, None, (f, None), rms=rms)
                assert (x == 2).all() and (q == (127 if rms else 0)).all()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_block_norm_most_rows(ops):
    """As many rows as the call takes: the last block's end is next to 2^31."""
    rows, C = 0x7fffff00, 8
    h = torch.ones(rows, C, dtype=BF16, device="cuda")
    gate, pre = torch.full((C,), 2.0, device="cuda"), (torch.ones(C, device="cuda"), torch.full((C,), 3.0, device="cuda"))
    x, y = ops.block_norm(h, gate=gate, pre=pre, out=h)
    assert x.data_ptr() == h.data_ptr()
    for lo in range(0, rows, 1 << 26):
        assert (x[lo:lo + (1 << 26)] == 2).all() and (y[lo:lo + (1 << 26)] == 3).all(), lo

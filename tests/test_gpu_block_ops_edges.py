"""Block operators at widths, views, sizes and values that the calls accept and that are easily got wrong, against their
formulas in 64 bits (bounds and helpers as in test_gpu_block_ops)."""
import math
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_block_ops import BF16, F16, block64, call_grouped, gen, near, operands, ops, rand, rotary64  # noqa: F401  (ops: fixture)

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


# ------------------------------------------------------------------------------------------------ GELU over all numbers
def gelu_values(N):
    """Arguments from the middle to where fp32 ends, both signs, infinities and NaN in front."""
    v = torch.cat([torch.logspace(-3, 38, N // 2 - 2), torch.tensor([6.08, 6.09])]).repeat_interleave(2)
    v[1::2] *= -1
    v[:3] = torch.tensor([math.inf, -math.inf, math.nan])
    return v.cuda()


def near_gelu(got, x):
    """Within 5.1e-7 of the exact value and one rounding; infinities and NaN as they are."""
    x = x.double()
    want = torch.where(x == -math.inf, torch.zeros_like(x), x * torch.special.ndtr(x))
    top = torch.finfo(got.dtype).max
    over = want >= top * (1 + torch.finfo(got.dtype).eps / 4)        # rounds to infinity
    assert (got[over & ~x.isnan()] == math.inf).all() and (got.isnan() == x.isnan()).all()
    keep = want.abs() < top * 0.99
    near(got[keep], want[keep], torch.full_like(want, 5.1e-7)[keep])


@pytest.mark.parametrize("t", [BF16, F16, torch.int8])
@pytest.mark.parametrize("S,E,N,K", [(3, 2, 136, 64), (300, 2, 136, 64), (17000, 3, 2568, 1024)])
def test_grouped_gelu_over_all_numbers(ops, S, E, N, K, t):
    """Warp dot products, single CTAs and CTA pairs: rows of zeros leave the bias as GELU's argument."""
    g = gen(S)
    a, w, sa, sw = operands(g, t, S, E, N, K)
    a.zero_()
    bias = gelu_values(N).expand(E, N).contiguous()
    off = torch.tensor([0] + [S * (e + 1) // E for e in range(E)], dtype=torch.int32, device="cuda")
    got = call_grouped(ops, a, w, sa, sw, off, bias=bias, gelu=True)
    ops.check_status()
    near_gelu(got, bias[:1].expand(S, N))


def test_dense_gelu_over_all_numbers(ops):
    N, K = 256, 64
    bias = gelu_values(N)
    w = torch.ones(N, K, dtype=BF16, device="cuda")
    for M in (100, 20000):                               # single CTAs, CTA pairs
        near_gelu(ops.gemm_bf16(torch.zeros(M, K, dtype=BF16, device="cuda"), w, bias, gelu=True), bias.expand(M, N))
        near_gelu(ops.gemm_i8(torch.zeros(M, K, dtype=torch.int8, device="cuda"), torch.ones(M, device="cuda"), w.to(torch.int8),
                              torch.ones(N, device="cuda"), bias, gelu=True), bias.expand(M, N))
    wc, meta = ops.pack_sp24(torch.zeros(N, K, dtype=torch.int8, device="cuda"))
    near_gelu(ops.gemm_i8_sp24(torch.zeros(300, K, dtype=torch.int8, device="cuda"), torch.ones(300, device="cuda"), wc, meta,
                               torch.ones(N, device="cuda"), bias, gelu=True), bias.expand(300, N))
    # quantised rows: a large negative argument leaves the row's largest value, GELU(1) = 0.84134 = 215.4 / 256, alone
    for C in (1280, 5120):
        x = torch.ones(33, C, dtype=BF16, device="cuda")
        x[:, ::2] = -1e10
        q, s = ops.quant_rows_i8(x, gelu=True)
        assert torch.equal(s, torch.full_like(s, 215 / 256 / 127)) and (q[:, ::2] == 0).all() and (q[:, 1::2] == 127).all()
    ops.check_status()


# ------------------------------------------------------------------------------------------------ overlapping operands
def test_overlapping_outputs_are_refused(ops):
    g = gen(5)
    buf = rand(g, 40, 64, t=BF16)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    fr, f = ops.rotary_freqs(64)[0], torch.ones(64, device="cuda")
    slots, wt = torch.zeros(20, 2, dtype=torch.int32, device="cuda"), torch.ones(20, 2, device="cuda")
    w, flat = rand(g, 2, 64, 64, t=BF16), buf.view(-1)
    before = buf.clone()
    for call in (lambda: ops.block_norm(buf[:20], out=buf[1:21]), lambda: ops.block_norm(rand(g, 20, 64, t=BF16), buf[:20], out=buf[19:39]),
                 lambda: ops.block_norm_quant_i8(buf[:20], None, None, (f, None), out=buf[4:24]),
                 lambda: ops.block_norm(buf[:20, :32], out=buf[:20, 24:56]),
                 lambda: ops.rotary(buf[None, :20], i32(0), fr, out=buf[None, 3:23]),
                 lambda: ops.rotary(flat.as_strided((2, 10, 64), (640, 64, 1)), i32(0), fr, out=flat.as_strided((2, 10, 64), (64, 128, 1))),
                 lambda: ops.gemm_grouped(buf[:20], w, i32(0, 10, 20), out=buf[19:39]),
                 lambda: ops.gemm_grouped(rand(g, 20, 64, t=BF16), w, i32(0, 10, 20), out=w.view(128, 64)[100:120]),
                 lambda: ops.combine_topk(buf[:20], slots, wt, out=buf[19:39]),
                 lambda: ops.combine_topk(rand(g, 20, 64, t=BF16), slots, wt, residual=buf[:20], out=buf[1:21])):
        with pytest.raises(RuntimeError, match="bad argument"):
            call()
    assert torch.equal(buf, before)


def test_outputs_between_the_operands_rows(ops):
    """Views of one buffer that share no element are as good as separate tensors."""
    g = gen(6)
    S, C = 300, 64
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    buf = rand(g, S, 5 * C, t=BF16)
    a, b, out = buf[:, :C], buf[:, C:2 * C], buf[:, 3 * C:4 * C]
    rest = buf.clone()
    want, _ = ops.block_norm(a.contiguous(), b.contiguous())
    ops.block_norm(a, b, out=out)
    assert torch.equal(out, want)
    w, off = rand(g, 2, C, C, t=BF16), i32(0, 100, S)
    want = ops.gemm_grouped(a.contiguous(), w, off)
    ops.gemm_grouped(a, w, off, out=out)
    assert torch.equal(out, want)
    slots, wt = torch.randint(-1, S, (S, 2), generator=g, device="cuda", dtype=torch.int32), rand(g, S, 2)
    want = ops.combine_topk(a.contiguous(), slots, wt, residual=b.contiguous())
    ops.combine_topk(a, slots, wt, residual=b, out=out)
    assert torch.equal(out, want)
    heads = lambda n: buf.as_strided((2, S, 32), (32, 5 * C, 1), n * C)
    fr, _ = ops.rotary_freqs(32)
    want = ops.rotary(heads(0).contiguous(), torch.arange(S, device="cuda"), fr)
    ops.rotary(heads(0), torch.arange(S, device="cuda"), fr, out=heads(3))
    assert torch.equal(heads(3), want)
    rest[:, 3 * C:4 * C] = buf[:, 3 * C:4 * C]
    assert torch.equal(buf, rest)
    # rows of unlike pitch, one tensor between the other's rows
    full = rand(g, 2, 10, C, t=BF16)
    want, _ = ops.block_norm(full[:, 0].contiguous())
    ops.block_norm(full[:, 0], out=full[0, 3:5])
    assert torch.equal(full[0, 3:5], want)


# ------------------------------------------------------------------------------------------------ rotary widths
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(20, 20), (20, 8), (2, 2), (30, 16), (12, 12), (81, 40)])
def test_rotary_of_padded_rows(ops, d, rot, interleaved):
    """Widths that are no multiples of 8, in rows that start at multiples of 8: the result is laid out alike."""
    g = gen(d)
    pad = -(-d // 8) * 8 + 8
    pos = torch.randint(0, 5000, (35,), generator=g, device="cuda")
    freqs, _ = ops.rotary_freqs(rot)
    for x in (rand(g, 3, 70, pad, t=BF16)[..., :d], rand(g, 70, 3, pad, t=F16)[..., :d].transpose(0, 1)):
        got = ops.rotary(x, pos, freqs, interleaved=interleaved)
        assert got.shape == x.shape and (got.stride(0) < got.stride(1)) == (x.stride(0) < x.stride(1))
        want, slack = rotary64(x, pos, freqs, interleaved, 1.0)
        near(got, want, slack)
        assert torch.equal(got[..., rot:], x[..., rot:])
        own = rand(g, 3, 70, pad, t=x.dtype)
        ops.rotary(x, pos, freqs, interleaved=interleaved, out=own[..., :d])
        assert torch.equal(own[..., :d], got)


# ------------------------------------------------------------------------------------------------ few rows
def test_grouped_few_rows_have_no_tensor_maps(ops):
    """Up to eight rows are dot products: pitches that no tensor map takes (single rows, so nothing lies that far) are fine."""
    from segment_anything_fast_b200 import _lib
    g = gen(9)
    a, w, off = rand(g, 1, 64, t=BF16), rand(g, 2, 32, 64, t=BF16), torch.tensor([0, 0, 1], dtype=torch.int32, device="cuda")
    out = torch.zeros(1, 32, dtype=BF16, device="cuda")
    rc = _lib.load().samb_gemm_grouped(a.data_ptr(), 1 << 40, 1, None, w.data_ptr(), 64, 64 * 32, None, off.data_ptr(), out.data_ptr(),
                                       1 << 40, 1, 2, 32, 64, 0, 0, None, ops.status_word(a.device).data_ptr(),
                                       torch.cuda.current_stream().cuda_stream)
    assert rc == 0 and torch.equal(out, ops.gemm_grouped(a, w, off))
    ops.check_status()


# ------------------------------------------------------------------------------------------------ host threads
def test_first_calls_from_several_threads(ops):
    """ctypes lets go of the interpreter's lock: twelve threads make their first calls at once, each on its own stream."""
    code = """
import threading
import torch
from segment_anything_fast_b200 import ops
torch.manual_seed(0)
norms = [(torch.randn(5000, C, device="cuda").bfloat16(), torch.ones(C, device="cuda")) for C in (1280, 1536, 1792, 2048)]
a, w = torch.randn(17000, 512, device="cuda").bfloat16(), torch.randn(3, 2568, 512, device="cuda").bfloat16()
off = torch.tensor([0, 4000, 12000, 17000], dtype=torch.int32, device="cuda")
rows = torch.randperm(17000, device="cuda", dtype=torch.int32)
ops.status_word(a.device)
calls = [lambda h=h, f=f: ops.block_norm(h, h, pre=(f, None))[1] for h, f in norms] * 2
calls += [lambda: ops.gemm_grouped(a, w, off), lambda: ops.gemm_grouped(a, w, off, rows=rows)] * 2
got, gate = [None] * len(calls), threading.Barrier(len(calls))
streams = [torch.cuda.Stream() for _ in calls]
torch.cuda.synchronize()
def work(i):
    with torch.cuda.stream(streams[i]):
        gate.wait()
        got[i] = [calls[i]() for _ in range(5)]
threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
for t in threads: t.start()
for t in threads: t.join()
torch.cuda.synchronize()
ops.check_status()
for i, c in enumerate(calls):
    want = c()
    assert got[i] is not None and all(torch.equal(o, want) for o in got[i]), i
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]

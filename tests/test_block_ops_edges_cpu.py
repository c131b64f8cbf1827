"""Block operators without a GPU: what the package needs of torch, and calls that are refused before a launch."""
import math
import os
import random
import re
import subprocess
import sys
from fractions import Fraction

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_package_imports_without_cuda_in_torch():
    """A torch built without CUDA has no ``_cuda_getCurrentRawStream``: registries and oracles load there all the same,
    and the stream comes from the public call."""
    code = """
import torch
del torch._C._cuda_getCurrentRawStream
import segment_anything_fast_b200
from segment_anything_fast_b200 import ops
class Stream:
    cuda_stream = 77
torch.cuda.current_device = lambda: 1
torch.cuda.current_stream = lambda dev: Stream if dev == 1 else None
assert ops._stream() == 77
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


def test_grouped_warps_leave_their_roles_together():
    """A wait that runs out may do so for some lanes of a warp only.  In the roles that a whole warp walks, no lane may act
    on its own answer (the others would meet it in elect.sync or __syncwarp and wait for good): a wait's result is only
    kept, what is issued asks for it behind the election, and the way out is a vote."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "segment_anything_fast_b200", "csrc", "gemm_grouped.cu")).read())
    uses = re.findall(r"[^;{}]*\bwarp_wait\([^;]*;", text.split("tile_list", 1)[1])
    assert len(uses) == 6                                # W, gathered rows, twice the MMA warp's two
    for use in uses:
        assert re.fullmatch(r"ok = (ok && )?warp_wait\([^;]*\);", use.strip()), use
    assert text.count("if (elect_one() && ok)") == 4 and "__activemask" not in text
    assert len(re.findall(r"ok = __all_sync\(0xffffffffu, ok\)", text)) == 4
    for role in re.split(r"\bok = true;", text)[1:]:
        role = role.split("warp ==", 1)[0]
        if "warp_wait(" in role:
            assert role.rindex("__all_sync") > role.rindex("warp_wait(")
            assert not re.search(r"if \(!ok\)|\(!\(ok = warp_wait", role)


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up pointers: only where no kernel can be launched")
    from segment_anything_fast_b200 import _lib, build
    build.build()
    return _lib.load()


BAD = -1
FAR = 1 << 40                                            # where nothing else lies
MB = 1 << 20


def cells(at, s0, n0, s1, n1, width):
    """The 16-byte cells of a strided operand (everything in bytes)."""
    at = at + np.arange(n0)[:, None, None] * s0 + np.arange(n1)[None, :, None] * s1 + np.arange(0, width, 16)
    return set(at.reshape(-1).tolist())


def test_overlaps_are_refused_and_views_between_rows_are_not(lib):
    """Outputs against operands at every offset and pitch, by brute force.  (What is not refused stops at the missing GPU.)"""
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(3000):
        C, rows = 8 * rng.randint(1, 4), rng.randint(1, 5)
        lda, ldo = (C + 8 * rng.randint(0, 9) for _ in range(2))
        if rng.random() < 0.5:
            ldo = lda
        at = MB + 16 * rng.randint(-60, 60)
        if at == MB and rng.random() < 0.9:
            continue
        a, o = cells(MB, 0, 1, 2 * lda, rows, 2 * C), cells(at, 0, 1, 2 * ldo, rows, 2 * C)
        shared, same = bool(a & o), at == MB and lda == ldo
        norm = lib.samb_block_norm(MB, lda, None, 0, None, None, None, None, None, 0, 1.0, 1e-6, 0, 0, at, ldo, None, rows, C, None)
        res = lib.samb_block_norm(FAR, C, MB, lda, None, None, None, None, None, 0, 1.0, 1e-6, 0, 0, at, ldo, None, rows, C, None)
        y = lib.samb_block_norm(MB, lda, None, 0, None, None, FAR, None, None, 0, 1.0, 1e-6, 0, 0, FAR + MB, C, at, rows, C, None)
        comb = lib.samb_combine_topk(MB, lda, rows, FAR, FAR, None, 0, at, ldo, rows, 1, C, 0, None)
        add = lib.samb_combine_topk(FAR, C, rows, FAR, FAR, MB, lda, at, ldo, rows, 1, C, 0, None)
        prod = lib.samb_gemm_grouped(MB, lda, rows, None, FAR, C, C * C, None, FAR + MB, at, ldo, rows, 2, C, C, 0, 0, None, FAR, None)
        assert (norm == BAD) == (shared and not same) and (res == BAD) == (shared and not same) and (add == BAD) == (shared and not same)
        assert (comb == BAD) == shared and (prod == BAD) == shared
        assert (y == BAD) == (bool(a & cells(at, 0, 1, 2 * C, rows, 2 * C)) and not (at == MB and lda == C))
        seen[shared] += 1
    assert min(seen) > 300
    seen = [0, 0]
    for _ in range(3000):
        d, planes, rows = 8 * rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 4)
        pad = lambda: 8 * rng.randint(0, 6)
        def layout():
            if rng.random() < 0.5:
                rs = d + pad()
                return rows * rs + pad(), rs
            ps = d + pad()
            return ps, planes * ps + pad()
        (xp, xr), (op, orow) = layout(), layout()
        if rng.random() < 0.6:
            op, orow = xp, xr
        at = MB + 16 * rng.choice([0] + list(range(-90, 91)))
        rc = lib.samb_rotary(MB, xp, xr, FAR, 0, rows, 1, FAR, d, 0, 1.0, at, op, orow, planes, rows, d, 0, None)
        shared = bool(cells(MB, 2 * xp, planes, 2 * xr, rows, 2 * d) & cells(at, 2 * op, planes, 2 * orow, rows, 2 * d))
        assert (rc == BAD) == (shared and not (at == MB and (xp, xr) == (op, orow)))
        seen[shared] += 1
    assert min(seen) > 300


def test_outputs_over_small_operands_are_refused(lib):
    """Parameters, indexes, scales and scratch inside an output."""
    def norm(x=2 * MB, y=3 * MB, pg=FAR, pb=FAR, qg=FAR, qb=FAR, gate=FAR):
        return lib.samb_block_norm(MB, 64, None, 0, pg, pb, qg, qb, gate, 2, 1.0, 1e-6, 0, 0, x, 64, y, 6, 64, None)
    assert norm() != BAD
    for name in ("pg", "pb", "qg", "qb", "gate"):
        assert norm(**{name: 2 * MB + 16}) == BAD and norm(**{name: 3 * MB + 752}) == BAD and norm(**{name: 3 * MB + 768}) != BAD
    assert norm(gate=2 * MB - 512) != BAD and norm(gate=2 * MB - 496) == BAD and norm(y=2 * MB + 16) == BAD

    def quant(s):
        return lib.samb_block_norm_quant_i8(MB, 64, None, 0, None, None, FAR, None, None, 0, 1.0, 1e-6, 0, 2 * MB, 64, 3 * MB, s, 6, 64, None)
    assert quant(4 * MB) != BAD
    for s in (MB + 4, 2 * MB + 764, 3 * MB - 20, 3 * MB + 380, FAR + 252):
        assert quant(s) == BAD
    assert quant(3 * MB - 24) != BAD and quant(3 * MB + 384) != BAD

    def rot(pos=FAR, freqs=FAR, p64=0):
        return lib.samb_rotary(MB, 640, 64, pos, p64, 10, 1, freqs, 64, 0, 1.0, 2 * MB, 640, 64, 3, 10, 64, 0, None)
    assert rot() != BAD and rot(pos=2 * MB) == BAD and rot(freqs=2 * MB + 3832) == BAD and rot(freqs=2 * MB + 3840) != BAD
    assert rot(pos=2 * MB - 40) != BAD and rot(pos=2 * MB - 40, p64=1) == BAD

    def comb(slots=FAR, w=FAR):
        return lib.samb_combine_topk(MB, 64, 20, slots, w, None, 0, 2 * MB, 64, 10, 2, 64, 0, None)
    assert comb() != BAD and comb(slots=2 * MB + 1276) == BAD and comb(w=2 * MB - 76) == BAD and comb(w=2 * MB - 80) != BAD

    def prod(out=3 * MB, off=FAR, rows=FAR, bias=FAR, w=2 * MB, scr=None, S=200, N=32, ldo=32):
        return lib.samb_gemm_grouped(MB, 64, 100, rows, w, 64, 64 * N, bias, off, out, ldo, S, 4, N, 64, 0, 1, scr, FAR, None)
    assert prod() != BAD
    assert prod(off=3 * MB) == BAD and prod(rows=3 * MB - 796) == BAD and prod(bias=3 * MB + 12796) == BAD and prod(w=3 * MB - 4 * 4096 + 16) == BAD
    assert prod(w=3 * MB - 4 * 4096) != BAD
    # scratch counts where it is used
    assert prod(scr=3 * MB) != BAD
    big = dict(S=65536, N=5120, ldo=5120, w=1 << 36, bias=1 << 35, rows=1 << 34, out=1 << 38)
    lib_rows = lambda scr: lib.samb_gemm_grouped(MB, 1280, 100, big["rows"], big["w"], 1280, 1280 * 5120, big["bias"], FAR, big["out"], 5120,
                                                 65536, 4, 5120, 1280, 0, 1, scr, FAR, None)
    assert lib_rows(1 << 39) != BAD and lib_rows(big["out"] + 1600) == BAD and lib_rows(MB) == BAD and lib_rows(big["rows"] - 16) == BAD


def test_rotary_angle_keeps_the_bound_in_the_header():
    """The kernel's arithmetic for an angle (64-bit fixed point, top 32 bits, fp32), restated, against whole numbers."""
    text = open(os.path.join(ROOT, "include", "samb200.h")).read()
    bound = re.search(r"off by at most \(([^)]*)\) turns", text).group(1).replace("^", "**").replace("|position|", "Fraction(pos)")
    two_pi = Fraction(2 * 3141592653589793238462643383279502884197169399375105820974944592307816406286, 10 ** 75)
    inv, inv_low, one = 0.15915494309189535, -9.839338337591243e-18, 2.0 ** 64
    rng = random.Random(2)
    worst = 0.0
    for _ in range(5000):
        f, pos = math.exp(rng.uniform(-14.0, 1.5)), rng.randint(0, 1 << rng.choice([6, 20, 40]))
        hi = f * inv
        lo = float(Fraction(f) * Fraction(inv) - Fraction(hi)) + f * inv_low
        step = (int((hi - math.floor(hi)) * one) + int(lo * one)) % (1 << 64)
        turn = (pos * step % (1 << 64)) >> 32
        got = Fraction(float(np.float32(turn - (1 << 32) if turn >= 1 << 31 else turn))) / (1 << 32)
        err = (got - Fraction(f) / two_pi * pos) % 1
        err = min(err, 1 - err)
        allowed = eval(bound, {"Fraction": Fraction, "pos": pos})
        assert err <= allowed
        worst = max(worst, float(err / allowed))
    assert worst > 0.5                                   # and it says no more than it has to


def test_grouped_tensor_memory_goes_back_after_the_drain():
    """A kernel that gave up waits for its copies and products in flight before it returns tensor memory: between the
    drain by one warp and the release by another stands a barrier."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "segment_anything_fast_b200", "csrc", "gemm_grouped.cu")).read())
    ends = re.findall(r"drain_copies<STAGES>\(full_bar(.*?)tmem_dealloc", text, flags=re.S)
    assert len(ends) == 2 and all("__syncthreads()" in e or "cluster_sync_all()" in e for e in ends)

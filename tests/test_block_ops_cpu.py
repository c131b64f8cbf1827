"""Host side of the block operators (norms around a block, rotary positions, mixture of experts): refusals that need
no GPU, and the frequencies of stretched rotary positions."""
import math

import pytest
import torch

P = 4096           # a non-null, aligned "device pointer": these calls are refused before anything is launched
BAD, SHAPE, ALIGN = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    from segment_anything_fast_b200 import _lib, build
    build.build()
    return _lib.load()


def _norm(lib, h=P, ldh=64, r=2 * P, ldr=64, pg=P, pb=P, qg=P, qb=P, gate=None, gates=0, f16=0, x=3 * P, ldx=64, y=4 * P,
          rows=6, C=64):
    return lib.samb_block_norm(h, ldh, r, ldr, pg, pb, qg, qb, gate, gates, 1.0, 1e-6, f16, 0, x, ldx, y, rows, C, None)


@pytest.mark.parametrize("want,change", [
    (BAD, dict(h=None)), (BAD, dict(x=None)), (BAD, dict(rows=-1)), (BAD, dict(C=0)), (BAD, dict(pg=None)),
    (BAD, dict(qg=None)), (BAD, dict(y=None)), (BAD, dict(y=3 * P)), (BAD, dict(x=P, ldx=72)), (BAD, dict(x=2 * P, ldx=72)),
    (BAD, dict(y=P, ldh=72)), (BAD, dict(y=2 * P, ldr=72)),
    (SHAPE, dict(C=60)), (SHAPE, dict(C=8200, ldh=8200, ldr=8200, ldx=8200)), (SHAPE, dict(rows=(1 << 31) - 4)),
    (SHAPE, dict(ldh=56)), (SHAPE, dict(ldh=68)), (SHAPE, dict(ldr=60)), (SHAPE, dict(ldx=63)),
    (SHAPE, dict(gate=P, gates=4)), (SHAPE, dict(gate=P, gates=0)),
    (ALIGN, dict(h=P + 2)), (ALIGN, dict(gate=P + 4, gates=2)), (ALIGN, dict(y=5 * P + 8)), (ALIGN, dict(pg=P + 4))])
def test_block_norm_refusals(lib, want, change):
    assert _norm(lib, **change) == want


def test_block_norm_quant_refusals(lib):
    f = lib.samb_block_norm_quant_i8
    assert f(P, 64, None, 0, None, None, P, None, None, 0, 1.0, 1e-6, 0, 2 * P, 64, 3 * P, None, 6, 64, None) == BAD
    assert f(P, 64, None, 0, None, None, None, None, None, 0, 1.0, 1e-6, 0, 2 * P, 64, None, P, 6, 64, None) == BAD
    assert f(P, 64, None, 0, None, None, P, None, None, 0, 1.0, 1e-6, 0, 2 * P, 64, P, 4 * P, 6, 64, None) == BAD   # yq over h
    assert f(P, 64, None, 0, None, None, P, None, None, 0, 1.0, 1e-6, 0, 2 * P, 64, 3 * P, 4 * P + 2, 6, 64, None) == ALIGN


def _rot(lib, x=P, ps=640, rs=64, pos=P, p64=0, period=5, axes=1, freqs=P, rot=64, out=2 * P, ops=640, ors=64, planes=3, rows=10,
         d=64):
    return lib.samb_rotary(x, ps, rs, pos, p64, period, axes, freqs, rot, 0, 1.0, out, ops, ors, planes, rows, d, 0, None)


@pytest.mark.parametrize("want,change", [
    (BAD, dict(x=None)), (BAD, dict(pos=None)), (BAD, dict(freqs=None)), (BAD, dict(out=None)), (BAD, dict(axes=3)),
    (BAD, dict(axes=0)), (BAD, dict(rot=0)), (BAD, dict(d=0)), (BAD, dict(planes=-1)), (BAD, dict(out=P, ops=648)),
    (SHAPE, dict(rot=66)), (SHAPE, dict(rot=63)), (SHAPE, dict(rot=62, axes=2)), (SHAPE, dict(period=0)),
    (SHAPE, dict(period=4)), (SHAPE, dict(ors=32)), (SHAPE, dict(ops=64)), (SHAPE, dict(ops=0)),
    (SHAPE, dict(x=P, out=P, ps=0, ops=0)), (SHAPE, dict(rs=-64)), (SHAPE, dict(rows=1 << 31, period=1 << 31)),
    (ALIGN, dict(rs=68)), (ALIGN, dict(ops=644)), (ALIGN, dict(x=P + 2)), (ALIGN, dict(freqs=P + 4)),
    (ALIGN, dict(pos=P + 4, p64=1))])
def test_rotary_refusals(lib, want, change):
    assert _rot(lib, **change) == want


def _route(lib, x=P, ld=16, T=3000, E=16, k=2, ids=P, w=P, slots=P, rows=P, off=P, scratch=P):
    return lib.samb_route_topk(x, ld, None, T, E, k, 0, 1, 1.0, ids, w, slots, rows, off, scratch, None)


@pytest.mark.parametrize("want,change", [
    (BAD, dict(x=None)), (BAD, dict(off=None)), (BAD, dict(slots=None)), (BAD, dict(T=-1)), (BAD, dict(k=0)),
    (BAD, dict(scratch=None)), (SHAPE, dict(k=9)), (SHAPE, dict(E=513, ld=513)), (SHAPE, dict(ld=15)),
    (SHAPE, dict(E=1, k=2)), (SHAPE, dict(T=1 << 30)), (SHAPE, dict(T=(1 << 31) - 1, k=1)), (ALIGN, dict(ids=P + 2))])
def test_route_refusals(lib, want, change):
    assert _route(lib, **change) == want


def _grouped(lib, a=P, lda=64, m=100, rows=P, w=2 * P, ldw=64, ws=64 * 32, bias=P, off=P, out=3 * P, ldo=32, S=200, E=4, N=32, K=64,
             epi=1, st=P, scr=None):
    return lib.samb_gemm_grouped(a, lda, m, rows, w, ldw, ws, bias, off, out, ldo, S, E, N, K, 0, epi, scr, st, None)


@pytest.mark.parametrize("want,change", [
    (BAD, dict(a=None)), (BAD, dict(w=None)), (BAD, dict(off=None)), (BAD, dict(out=None)), (BAD, dict(st=None)),
    (BAD, dict(bias=None)), (BAD, dict(epi=0)), (BAD, dict(epi=4 + 1)), (BAD, dict(epi=8)), (BAD, dict(S=-1)),
    (BAD, dict(m=0)), (BAD, dict(E=0)), (BAD, dict(out=P)), (BAD, dict(out=2 * P)),
    (SHAPE, dict(N=36, ldo=40)), (SHAPE, dict(K=60)), (SHAPE, dict(lda=56)), (SHAPE, dict(ldw=60)), (SHAPE, dict(ldo=24)),
    (SHAPE, dict(ws=64 * 16)), (SHAPE, dict(rows=None)), (SHAPE, dict(E=513)), (SHAPE, dict(S=(1 << 31) - 1)),
    (SHAPE, dict(S=(1 << 31) - 200, N=1 << 20, ldo=1 << 20, ws=1 << 26)),
    (ALIGN, dict(a=P + 8)), (ALIGN, dict(scr=P + 8)), (ALIGN, dict(out=P + 2)), (ALIGN, dict(off=P + 1)), (ALIGN, dict(rows=P + 2))])
def test_grouped_refusals(lib, want, change):
    assert _grouped(lib, **change) == want


def test_grouped_i8_refusals(lib):
    def call(scale=P, ws=P, K=64):
        return lib.samb_gemm_i8_grouped(P, 64, 100, scale, P, 2 * P, 64, 64 * 32, ws, None, P, 3 * P, 32, 200, 4, 32, K, 0, None, P, None)
    assert call(scale=None) == BAD and call(ws=None) == BAD
    assert call(K=56) == SHAPE                       # 8-element steps are enough for 16-bit types only


def _combine(lib, x=P, ldx=64, n=20, slots=P, w=P, r=2 * P, ldr=64, out=3 * P, ldo=64, T=10, k=2, C=64):
    return lib.samb_combine_topk(x, ldx, n, slots, w, r, ldr, out, ldo, T, k, C, 0, None)


@pytest.mark.parametrize("want,change", [
    (BAD, dict(x=None)), (BAD, dict(slots=None)), (BAD, dict(w=None)), (BAD, dict(out=None)), (BAD, dict(out=P)),
    (BAD, dict(T=-1)), (BAD, dict(k=0)), (BAD, dict(out=2 * P, ldo=72)), (SHAPE, dict(k=9)), (SHAPE, dict(C=60)),
    (SHAPE, dict(ldx=56)), (SHAPE, dict(ldr=68)), (SHAPE, dict(T=1 << 31)), (ALIGN, dict(x=P + 4)), (ALIGN, dict(slots=P + 2))])
def test_combine_refusals(lib, want, change):
    assert _combine(lib, **change) == want


def test_argument_types_match_the_header():
    """Every argument of every function, as the header declares it, against the ctypes table."""
    import ctypes
    import os
    import re
    from segment_anything_fast_b200 import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(root, "include", "samb200.h")).read(), flags=re.S)
    plain = {"int": ctypes.c_int, "int32_t": ctypes.c_int32, "uint32_t": ctypes.c_uint32, "int64_t": ctypes.c_int64,
             "float": ctypes.c_float}
    seen = 0
    for name, args in re.findall(r"\b(samb_[a-z0-9_]+)\s*\(([^)]*)\)", text):
        want = [] if args.strip() == "void" else [a.strip() for a in args.split(",")]
        have = _lib.SIGNATURES[name][1]
        assert len(want) == len(have), name
        for w, h in zip(want, have):
            if "*" in w:
                assert h is ctypes.c_void_p or issubclass(h, ctypes._Pointer), (name, w)
            else:
                assert h is plain[w.replace("const ", "").split()[0]], (name, w)
        seen += 1
    assert seen == len(_lib.SIGNATURES)


def test_wrappers_refuse_cpu_tensors():
    from segment_anything_fast_b200 import ops
    h = torch.zeros(4, 64, dtype=torch.bfloat16)
    i = torch.zeros(5, dtype=torch.int32)
    f = torch.zeros(4, 4)
    for call in (lambda: ops.block_norm(h), lambda: ops.block_norm_quant_i8(h, None, None, (f, None)),
                 lambda: ops.rotary(h[None], i[:4], torch.zeros(32, dtype=torch.float64)),
                 lambda: ops.route_topk(f, 2), lambda: ops.gemm_grouped(h, h[None], i),
                 lambda: ops.gemm_i8_grouped(h.to(torch.int8), f, h[None].to(torch.int8), f, i),
                 lambda: ops.combine_topk(h, i[:4].reshape(2, 2), f)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_rotary_freqs():
    from segment_anything_fast_b200 import ops
    cpu = torch.device("cpu")
    f, m = ops.rotary_freqs(8, device=cpu)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, _ = ops.rotary_freqs(16, axes=2, device=cpu)                       # four pairs an axis, the same on both
    assert torch.equal(g[:4], f) and torch.equal(g[4:], f)
    assert torch.allclose(ops.rotary_freqs(8, scaling="linear", factor=4.0, device=cpu)[0], f / 4, rtol=1e-14)
    b, _ = ops.rotary_freqs(8, scaling="base", factor=4.0, device=cpu)
    assert b[0] == 1.0 and math.isclose(b[-1], f[-1] / 4, rel_tol=1e-12)
    p, m = ops.rotary_freqs(8, scaling="parts", factor=4.0, trained=1000, device=cpu)
    assert math.isclose(m, 0.1 * math.log(4.0) + 1)
    assert p[0] == f[0] and math.isclose(p[3], f[3] / 4, rel_tol=1e-12)    # 159 turns are kept, 0.16 are stretched
    keep = (1000 * 0.1 / (2 * math.pi) - 1) / 31                           # 15.9 turns: on the ramp
    assert math.isclose(p[1], 0.1 * (keep + (1 - keep) / 4), rel_tol=1e-12)
    for bad in (dict(rot=7), dict(rot=6, axes=2), dict(rot=0), dict(rot=8, scaling="other"), dict(rot=8, factor=0.5),
                dict(rot=8, axes=3), dict(rot=8, base=0.0)):
        with pytest.raises(RuntimeError):
            ops.rotary_freqs(device=cpu, **bad)


def test_grouped_scratch(lib):
    f = lib.samb_gemm_grouped_scratch_bytes
    assert f(2, 16, 5120, 1280, 0) == f(0, 1, 5120, 64, 0) == f(511 * 16, 16, 5120, 1280, 0) == f(65536, 16, 1280, 5120, 0) == 0
    assert f(65536, 16, 5120, 1280, 0) == 65536 * 1280 * 2 and f(1 << 30, 8, 5120, 5120, 1) == 5120 << 30


def test_route_scratch(lib):
    assert lib.samb_route_scratch_bytes(1, 16) == 0 and lib.samb_route_scratch_bytes(0, 16) == 0
    assert lib.samb_route_scratch_bytes(1 << 20, 512) == 148 * 512 * 4
    assert lib.samb_route_scratch_bytes(-1, 16) == 0 and lib.samb_route_scratch_bytes(10, 513) == 0

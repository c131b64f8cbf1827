"""The block operators (norms around a block, rotary positions, mixture of experts) against their formulas in 64 bits.

Tolerances: an output is the exact value, plus the fp32 arithmetic's error (bounded below per operator from the number
of roundings in the longest chain, 2^-24 each, times the sum of the absolute terms), rounded once to its type
(``finfo.eps / 2`` relative)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
U32 = 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from segment_anything_fast_b200 import ops as _ops
    return _ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, by=1.0, at=0.0, t=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * by + at).to(t)


def near(got, want, slack):
    """|got - want| <= half a step of got's type, relative to what is rounded, plus slack."""
    err = (got.double() - want).abs()
    # the smallest step of a subnormal float16 (2^-24) may be the half step there
    bound = (want.abs() + slack) * (torch.finfo(got.dtype).eps / 2) + slack + (2.0 ** -25 if got.dtype == F16 else 0.0)
    bad = ~(err <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst by {float((err - bound).max()):.3g} at {bad.nonzero()[0].tolist()}"


# ------------------------------------------------------------------------------------------------ block_norm
def norm64(v, affine, rms, err):
    """The norm of v in 64 bits and a bound on the fp32 form's error; err: bound on the error that v comes with.
    Chains: 8 elements a thread, 5 shuffle steps, up to 32 warps, then mean, deviation, product, offset: under 64
    roundings.  An error d in v moves the normalised value by d * rstd on its own and, through mean and variance, by at
    most the row's largest d * rstd times (1 + |z|) twice."""
    if affine is None:
        return v, err
    g, b = affine
    mean = v.mean(1, keepdim=True) if not rms else torch.zeros_like(v[:, :1])
    c = v - mean
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-6)
    z = c * rstd
    out = z * g.double() + (b.double() if b is not None else 0.0)
    # the mean is off by 64 roundings of the mean absolute value, the deviation by that and its own rounding
    d = err + 64 * U32 * (v.abs().mean(1, keepdim=True) + v.abs())
    dm = d.amax(1, keepdim=True)
    e = (d + dm) * rstd + z.abs() * (dm * rstd + 64 * U32)
    return out, e * g.double().abs() + 4 * U32 * (z * g.double()).abs() + (4 * U32 * b.double().abs() if b is not None else 0.0)


def block64(h, r, post, pre, gate, a, rms):
    u, e = norm64(h.double(), post, rms, torch.zeros_like(h, dtype=torch.float64))
    if gate is not None:
        gt = gate.double().reshape(-1, h.shape[1]).repeat_interleave(h.shape[0] // (gate.numel() // h.shape[1]), 0)
        u, e = u * gt, e * gt.abs() + 4 * U32 * (u * gt).abs()
        if post is not None and post[1] is not None:     # gain and offset are multiplied by the gate first
            e = e + 4 * U32 * (post[1].double() * gt).abs() + 4 * U32 * (u - post[1].double() * gt).abs()
    x = u + (a * r.double() if r is not None else 0.0)
    e = e + 4 * U32 * (u.abs() + (abs(a) * r.double().abs() if r is not None else 0.0))
    y, ey = norm64(x, pre, rms, e)
    return x, e, y, ey


@pytest.mark.parametrize("t,rms", [(BF16, False), (BF16, True), (F16, False), (F16, True)])
@pytest.mark.parametrize("rows,C,gates", [(1, 8, 0), (1, 1280, 1), (3, 256, 3), (5, 264, 0), (7, 1280, 7), (130, 200, 2), (1031, 768, 1),
                                          (6000, 1280, 6), (2376, 2048, 24), (2, 2056, 2), (300, 4104, 3), (151, 8192, 0),
                                          (60000, 64, 8), (39999, 256, 3), (30011, 264, 1)])
def test_block_norm(ops, rows, C, gates, t, rms):
    g = gen(rows * 7 + C)
    h, r = rand(g, rows, C, at=0.3, t=t), rand(g, rows, C, by=3.0, t=t)
    post = (rand(g, C, by=0.2, at=1.0), None if rms else rand(g, C))
    pre = (rand(g, C, by=0.2, at=1.0), None if rms else rand(g, C))
    gate = None if gates == 0 else rand(g, C) if gates == 1 else rand(g, gates, C)
    x, y = ops.block_norm(h, r, post=post, pre=pre, gate=gate, res_scale=0.75, rms=rms)
    x64, ex, y64, ey = block64(h, r, post, pre, gate, 0.75, rms)
    near(x, x64, ex)
    near(y, y64, ey)


@pytest.mark.parametrize("C", [256, 1280, 2304])
@pytest.mark.parametrize("post,pre,res,gate", [(0, 0, 1, 1), (1, 0, 1, 0), (0, 1, 1, 0), (0, 1, 0, 1), (1, 1, 0, 0)])
def test_block_norm_parts_left_out(ops, C, post, pre, res, gate):
    g = gen(C + post * 8 + pre * 4 + res * 2 + gate)
    h, r = rand(g, 777, C, t=BF16), rand(g, 777, C, t=BF16) if res else None
    post = (rand(g, C), rand(g, C)) if post else None
    pre = (rand(g, C), rand(g, C)) if pre else None
    gate = rand(g, 7, C) if gate else None
    x, y = ops.block_norm(h, r, post=post, pre=pre, gate=gate)
    x64, ex, y64, ey = block64(h, r, post, pre, gate, 1.0, False)
    near(x, x64, ex)
    assert (y is None) == (pre is None)
    if pre is not None:
        near(y, y64, ey)


def test_block_norm_in_place_and_strided(ops):
    g = gen(3)
    wide, wider = rand(g, 4099, 1536, t=BF16), rand(g, 4099, 1312, t=BF16)
    h, r = wide[:, 128:1408], wider[:, 16:1296]
    pre = (rand(g, 1280), rand(g, 1280))
    want, wanty = ops.block_norm(h.contiguous(), r.contiguous(), post=pre, pre=pre)
    around = wider.clone()
    x, y = ops.block_norm(h, r, post=pre, pre=pre, out=r)
    assert x.data_ptr() == r.data_ptr() and torch.equal(r, want) and torch.equal(y, wanty)
    assert torch.equal(wider[:, :16], around[:, :16]) and torch.equal(wider[:, 1296:], around[:, 1296:])
    h2 = h.contiguous()
    x, y = ops.block_norm(h2, around[:, 16:1296], post=pre, pre=pre, out=h2)
    assert torch.equal(h2, want) and torch.equal(y, wanty)


def test_block_norm_hard_rows(ops):
    """A constant row, a row far from zero, rows with an infinity or a NaN: nobody else's row notices."""
    g = gen(4)
    h = rand(g, 64, 1280, t=BF16)
    r = torch.zeros_like(h)
    pre = (torch.ones(1280, device="cuda"), torch.zeros(1280, device="cuda"))
    clean = ops.block_norm(h, r, post=pre, pre=pre)
    h[3] = 2.0
    h[10] = (256 + rand(g, 1280)).to(BF16)
    h[20, 7], h[21, 1279] = math.inf, math.nan
    x, y = ops.block_norm(h, r, post=pre, pre=pre)
    assert torch.equal(x[3], torch.zeros_like(x[3]))     # deviations from the mean are exactly 0
    x64, ex, y64, ey = block64(h, r, pre, pre, None, 1.0, False)
    near(x[10:11], x64[10:11], ex[10:11])
    assert x[20].isnan().all() and x[21].isnan().all()   # inf - inf, and NaN
    keep = torch.ones(64, dtype=torch.bool, device="cuda")
    keep[[3, 10, 20, 21]] = False
    assert torch.equal(x[keep], clean[0][keep]) and torch.equal(y[keep], clean[1][keep])


@pytest.mark.parametrize("rows,C,rms", [(1, 1280, False), (777, 256, False), (6003, 1280, False), (515, 1280, True), (65, 4096, False)])
def test_block_norm_quant(ops, rows, C, rms):
    g = gen(rows + C)
    h, r = rand(g, rows, C, t=BF16), rand(g, rows, C, t=BF16)
    h[rows // 2] = 0
    r[rows // 2] = 0
    post, pre = (rand(g, C), None if rms else rand(g, C)), (rand(g, C), None)
    gate = rand(g, C)
    gate = gate if rms else gate * 0.5
    x, yq, s = ops.block_norm_quant_i8(h, r, post, pre, gate=gate, rms=rms)
    x2, y2 = ops.block_norm(h, r, post, pre, gate=gate, rms=rms)
    q2, s2 = ops.quant_rows_i8(y2)
    assert torch.equal(x, x2) and torch.equal(s, s2) and torch.equal(yq, q2)


# ------------------------------------------------------------------------------------------------ rotary
def rotary64(x, positions, freqs, interleaved, mscale):
    half = freqs.numel()
    pos = positions.reshape(positions.shape[0], -1)
    axes = pos.shape[1]
    # the angle modulo one turn from whole-number arithmetic: frequency / 2 pi to 128 bits
    two_pi = 2 * 3141592653589793238462643383279502884197169399375105820974944592307816406286
    one = 10 ** 75
    steps = []
    for f in freqs.tolist():
        m, e = math.frexp(f)
        m = int(m * 2 ** 53)
        steps.append(((m << 128) * one * 2 ** max(0, e - 53)) // (two_pi * 2 ** max(0, 53 - e)))
    ang = torch.empty(pos.shape[0], half, dtype=torch.float64)
    pl = pos.cpu().tolist()
    for i, row in enumerate(pl):
        for j in range(half):
            t = (row[j * axes // half] * steps[j]) % (1 << 128)
            ang[i, j] = 2 * math.pi * (t / 2.0 ** 128)
    ang = ang.cuda().repeat(x.shape[1] // pos.shape[0], 1)
    c, s = ang.cos() * mscale, ang.sin() * mscale
    out = x.double().clone()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else (x[..., :half], x[..., half:2 * half])
    a, b = a.double(), b.double()
    lo, hi = a * c - b * s, b * c + a * s
    # angle: 2^-32 turns and its fp32 rounding (2^-24 of half a turn); sincospi within 2 units of 2^-24; product, sum
    slack = torch.zeros_like(out)
    e = (a.abs() + b.abs()) * mscale * (math.pi * 2.0 ** -24 + 2 * math.pi * 2.0 ** -32 + 8 * U32)
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = lo, hi
        slack[..., 0:2 * half:2], slack[..., 1:2 * half:2] = e, e
    else:
        out[..., :half], out[..., half:2 * half] = lo, hi
        slack[..., :half], slack[..., half:2 * half] = e, e
    return out, slack


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("planes,rows,d,rot,axes,period,far", [
    (1, 1, 8, 2, 1, 1, 0), (32, 1, 80, 80, 1, 1, 1000000), (4, 64, 64, 64, 2, 64, 64), (3, 35, 80, 80, 2, 7, 300),
    (2, 130, 80, 40, 1, 130, 4096), (5, 33, 128, 36, 2, 11, 77), (7, 12, 24, 22, 1, 4, 50000), (2, 9, 16, 16, 1, 9, 1 << 40),
    (1, 3000, 256, 128, 1, 1000, 1 << 30), (40, 17, 32, 4, 2, 17, 5), (1, 70000, 16, 8, 1, 1, 9), (3, 5000, 24, 24, 1, 2, 31)])
def test_rotary(ops, planes, rows, d, rot, axes, period, far, interleaved, t):
    g = gen(planes * 31 + rows + rot)
    x = rand(g, planes, rows, d, t=t)
    pos = torch.randint(0, far + 1, (period, 2) if axes == 2 else (period,), generator=g, device="cuda")
    pos[-1] = far
    freqs, m = ops.rotary_freqs(rot, axes=axes, scaling="parts" if far > 4096 else None, factor=4.0)
    got = ops.rotary(x, pos, freqs, interleaved=interleaved, mscale=m)
    want, slack = rotary64(x, pos, freqs, interleaved, m)
    near(got, want, slack)
    assert torch.equal(got[..., rot:], x[..., rot:])
    if far < 1 << 31:
        assert torch.equal(ops.rotary(x, pos.int(), freqs, interleaved=interleaved, mscale=m), got)


def test_rotary_turns_back(ops):
    """Position -p undoes position p; negative frequencies are the same as negative positions."""
    g = gen(8)
    x = rand(g, 4, 50, 64, t=BF16)
    pos = torch.randint(1, 100000, (50,), generator=g, device="cuda")
    freqs, _ = ops.rotary_freqs(64)
    back, slack = rotary64(x, -pos, freqs, False, 1.0)
    near(ops.rotary(x, -pos, freqs), back, slack)
    near(ops.rotary(x, pos, -freqs), back, slack)
    assert torch.equal(ops.rotary(x, torch.zeros_like(pos), freqs), x)


@pytest.mark.parametrize("rot", [80, 48])
def test_rotary_views_and_in_place(ops, rot):
    g = gen(9)
    qkv = rand(g, 48, 200, 80, t=BF16)
    freqs, _ = ops.rotary_freqs(rot, axes=2)
    pos = torch.stack([torch.arange(100) % 10, torch.arange(100) // 10], 1).cuda()
    want = ops.rotary(qkv[:32].contiguous(), pos, freqs)
    work = qkv.clone()
    assert ops.rotary(work[:32], pos, freqs, out=work[:32]).data_ptr() == work.data_ptr()
    assert torch.equal(work[:32], want) and torch.equal(work[32:], qkv[32:])
    # token-major rows of 16 heads in a wider buffer: only the heads' own elements change
    tok = torch.zeros(200, 16 * 80 + 64, dtype=BF16, device="cuda")
    tok[:, :1280] = qkv[:16].transpose(0, 1).reshape(200, 1280)
    view = tok.as_strided((16, 200, 80), (80, 1344, 1))
    ops.rotary(view, pos, freqs, out=view)
    assert torch.equal(view, want[:16]) and (tok[:, 1280:] == 0).all()
    back = torch.empty(200, 16, 80, dtype=BF16, device="cuda")
    ops.rotary(qkv[:16], pos, freqs, out=back.transpose(0, 1))
    assert torch.equal(back.transpose(0, 1), want[:16])


# ------------------------------------------------------------------------------------------------ router
def route_plain(x, k, bias, sigmoid, renorm, scale):
    x = torch.where(x.isnan(), torch.full_like(x, -math.inf), x).clamp(max=torch.finfo(torch.float32).max)
    T, E = x.shape
    key = x if bias is None else x + bias
    key = torch.where((x == -math.inf) | key.isnan(), torch.full_like(x, -math.inf), key)
    top, ids = torch.sort(key, dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k]
    x64 = x.double()
    hi = x64.amax(1, keepdim=True).clamp(min=-1e300)
    p = torch.sigmoid(x64) if sigmoid else torch.exp(x64 - hi)
    if not sigmoid:
        p = p / p.sum(1, keepdim=True)
    w = torch.where(top == -math.inf, torch.zeros_like(p[:, :k]), p.gather(1, ids))
    dist = (x64.gather(1, ids) - hi).abs() if not sigmoid else x64.gather(1, ids).abs()
    if renorm:                                           # of logarithms: even in 64 bits exp and sigmoid can vanish
        lw = (torch.nn.functional.logsigmoid(x64) if sigmoid else x64).gather(1, ids)
        w = torch.softmax(torch.where(top == -math.inf, torch.full_like(lw, -math.inf), lw), 1).nan_to_num(0.0)
    ids = torch.where(top == -math.inf, torch.full_like(ids, -1), ids)
    flat = torch.where(ids < 0, torch.full_like(ids, E), ids).reshape(-1)
    by, order = torch.sort(flat, stable=True)
    off = torch.searchsorted(by, torch.arange(E + 1, device=x.device))
    at = torch.arange(T * k, device=x.device)
    slots = torch.empty_like(order)
    slots[order] = torch.where(by < E, at, torch.full_like(at, -1))
    rows = torch.where(by < E, order // k, torch.full_like(order, -1))
    return ids, w * scale, slots.reshape(T, k), rows, off, dist


def check_route(ops, x, k, bias=None, sigmoid=False, renorm=True, scale=1.0):
    r = ops.route_topk(x, k, bias=bias, sigmoid=sigmoid, renorm=renorm, scale=scale)
    ids, w, slots, rows, off, dist = route_plain(x, k, bias, sigmoid, renorm, scale)
    for got, want, name in ((r.ids, ids, "ids"), (r.slots, slots, "slots"), (r.rows, rows, "rows"), (r.offsets, off, "offsets")):
        assert torch.equal(got.long(), want), name
    # exp of a difference d rounded to fp32 is off by d 2^-24 relative, expf by 2 units; the sum takes 16 + 5 steps and
    # the renormalising one 8; a weight below the least normal float may go to zero
    tol = w.abs() * (2 * dist.clamp(max=200) + 64) * U32 + 2.0 ** -120
    if renorm:
        tol = w.abs() * (2 * dist.clamp(max=200) + 2 * dist[:, :1].clamp(max=200) + 96) * U32 + 2.0 ** -120
    assert ((r.weights.double() - w).abs() <= tol).all()
    return r


@pytest.mark.parametrize("sigmoid,renorm", [(False, True), (False, False), (True, True), (True, False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 16, 2), (2, 3, 3), (31, 33, 8), (128, 64, 4), (129, 64, 4), (32, 65, 3), (33, 65, 3), (1000, 130, 6),
                                   (2369, 8, 2), (5000, 512, 8), (40000, 16, 1)])
def test_route(ops, T, E, k, sigmoid, renorm):
    g = gen(T + E)
    x = rand(g, T, E, by=2.0)
    check_route(ops, x, k, None, sigmoid, renorm, 2.5)
    tied = (x * 2).round() / 2                                             # few different values: ties everywhere
    tied[torch.rand(T, E, generator=g, device="cuda") < 0.3] = -math.inf
    tied[T // 2:T // 2 + 5] = -math.inf
    check_route(ops, tied, k, rand(g, E).round(), sigmoid, renorm)


def test_route_hard_values(ops):
    inf, nan, low = math.inf, math.nan, torch.finfo(torch.float32).min
    x = torch.tensor([[0.0, -0.0, 0.0, -0.0], [inf, 1.0, inf, 0.0], [nan, -inf, 2.0, nan], [low, low, low, low],
                      [low, low, 3.0, -inf], [-inf, -inf, -inf, -inf], [nan, nan, nan, nan], [1e38, -1e38, 3e38, 0.0],
                      [88.0, -88.0, 500.0, -500.0]], device="cuda")
    r = check_route(ops, x, 2)
    assert r.ids.tolist() == [[0, 1], [0, 2], [2, -1], [0, 1], [2, 0], [-1, -1], [-1, -1], [2, 0], [2, 0]]
    assert r.weights[:5].tolist() == [[0.5, 0.5], [0.5, 0.5], [1.0, 0.0], [0.5, 0.5], [1.0, 0.0]]
    assert not r.weights.isnan().any()
    check_route(ops, x, 3, sigmoid=True)
    check_route(ops, x, 4, bias=torch.tensor([0.0, 5.0, -inf, nan], device="cuda"))


def test_route_strided_and_empty(ops):
    g = gen(5)
    wide = rand(g, 700, 96)
    r, want = ops.route_topk(wide[:, 16:48], 2), ops.route_topk(wide[:, 16:48].contiguous(), 2)
    for a, b in zip(r, want):
        assert torch.equal(a, b)
    r.ids.fill_(5)                                       # the results are ordinary tensors, apart from one another
    assert torch.equal(r.slots, want.slots) and torch.equal(r.rows, want.rows) and torch.equal(r.offsets, want.offsets)
    r = ops.route_topk(wide[:0, :8], 2)
    assert r.ids.shape == (0, 2) and r.rows.numel() == 0 and r.offsets.tolist() == [0] * 9


@pytest.mark.parametrize("T,E,k", [(5, 16, 2), (300, 24, 3), (1000, 64, 8), (129, 60, 5), (200, 128, 4)])
def test_route_whatever_the_alignment(ops, T, E, k):
    """Rows that start off 16-byte boundaries, an odd pitch, a bias off its boundary: the same results."""
    g = gen(T * E)
    x, b = (2 * rand(g, T, E)).round(), rand(g, E).round()
    want = ops.route_topk(x, k, bias=b)
    check_route(ops, x, k, b)
    flat = torch.zeros(T * (E + 9) + 1, device="cuda")
    off_bias = torch.empty(E + 1, device="cuda")[1:].copy_(b)
    for pitch, first in ((E + 8, 0), (E + 8, 1), (E + 9, 0), (E, 1)):
        view = flat.as_strided((T, E), (pitch, 1), first).copy_(x)
        for bias in (b, off_bias):
            for p, q in zip(ops.route_topk(view, k, bias=bias), want):
                assert torch.equal(p, q)


# ------------------------------------------------------------------------------------------------ grouped products
def grouped64(a, w, offsets, rows, bias, gelu, S, a_scale=None, w_scale=None):
    """Outputs, slack and which rows are written.  fp32 accumulation in the tensor core: K products, each addition off
    by at most 2^-23 of the partial sum; int8 sums are exact and scaled by two products; GELU is within 5.1e-7 of
    exact and has a slope below 1.13."""
    E, N, K = w.shape
    out = torch.zeros(S, N, dtype=torch.float64, device=a.device)
    slack = torch.zeros_like(out)
    written = torch.zeros(S, dtype=torch.bool, device=a.device)
    o = offsets.tolist()
    for e in range(E):
        lo, hi = o[e], o[e + 1]
        if hi <= lo:
            continue
        src = torch.arange(lo, hi, device=a.device) if rows is None else rows[lo:hi].long()
        ok = (src >= 0) & (src < a.shape[0])
        ae = torch.where(ok[:, None], a[src.clamp(0, a.shape[0] - 1)].double(), torch.zeros((), dtype=torch.float64, device=a.device))
        y, mag = ae @ w[e].double().t(), ae.abs() @ w[e].double().abs().t()
        if a_scale is not None:
            s = a_scale[src.clamp(0, a.shape[0] - 1)].double()[:, None] * w_scale[e].double()
            y, err = y * s, 3 * U32 * (y * s).abs()
        else:
            err = K * 2.0 ** -23 * mag
        if bias is not None:
            y = y + bias[e].double()
            err = err + U32 * y.abs()
        if gelu:
            y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
            err = 1.13 * err + 6e-7 + 4 * U32 * y.abs()
        out[lo:hi], slack[lo:hi], written[lo:hi] = y, err, True
    return out, slack, written


def operands(g, t, M, E, N, K, pad=0):
    if t == torch.int8:
        a = torch.randint(-127, 128, (M, K + 16 * pad), generator=g, device="cuda", dtype=torch.int8)[:, :K]
        w = torch.randint(-127, 128, (E, N + pad, K + 16 * pad), generator=g, device="cuda", dtype=torch.int8)[:, :N, :K]
        sa = torch.rand(M, generator=g, device="cuda") * 0.02 + 0.001
        sw = torch.rand(E, N, generator=g, device="cuda") * 0.01 / math.sqrt(K) + 1e-4
        return a, w, sa, sw
    a = rand(g, M, K + 8 * pad, t=t)[:, :K]
    w = rand(g, E, N + pad, K + 8 * pad, by=1 / math.sqrt(K), t=t)[:, :N, :K]
    return a, w, None, None


def call_grouped(ops, a, w, sa, sw, off, **kw):
    if a.dtype == torch.int8:
        return ops.gemm_i8_grouped(a, sa, w, sw, off, **kw)
    return ops.gemm_grouped(a, w, off, **kw)


CASES = [  # counts of the experts, rows behind the last, N, K, padded strides
    ([1], 0, 8, 16, 0), ([1, 1], 0, 256, 64, 0), ([0, 2, 0, 1, 0], 3, 264, 80, 0), ([127, 128, 129], 0, 256, 320, 0),
    ([0, 0, 300, 0], 5, 520, 64, 0), ([5, 260, 1, 0, 64], 0, 72, 144, 1), ([1] * 33, 2, 64, 96, 0), ([3] * 300, 0, 40, 32, 0),
    ([700, 11, 90], 0, 1280, 1280, 0), ([1] * 8, 0, 1280, 5120, 0), ([8, 0, 3], 1, 640, 1296, 1), ([2] * 16, 0, 2560, 256, 0),
    ([4000, 3000, 1192], 0, 1288, 128, 0), ([9000, 3, 4570], 5, 1032, 528, 1), ([20000, 0], 7, 520, 512, 0), ([600], 0, 8, 16, 0),
    ([9000, 7001, 0, 700], 9, 2568, 528, 0),
    ([100, 40, 0, 200], 0, 256, 1040, 0), ([0] * 250 + [3] + [0] * 200 + [2] + [0] * 58, 1, 264, 64, 0), ([2, 0, 1] * 170 + [1, 1], 3, 40, 32, 0)]


@pytest.mark.parametrize("t", [BF16, F16, torch.int8])
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("counts,behind,N,K,pad", CASES)
def test_gemm_grouped(ops, counts, behind, N, K, pad, gather, t):
    g = gen(sum(counts) + N + K)
    S, E = sum(counts) + behind, len(counts)
    off = torch.tensor([0] + counts, device="cuda").cumsum(0).int()
    M = max(1, S // 2) if gather else S
    a, w, sa, sw = operands(g, t, M, E, N, K, pad)
    rows = torch.randint(0, M, (S,), generator=g, device="cuda", dtype=torch.int32) if gather else None
    bias = rand(g, E, N)
    ot = BF16 if t == torch.int8 else t
    for b, gelu in ((None, False), (bias, True), (bias, False)):
        buf = torch.full((S + 2, N + 24), 7.0, dtype=ot, device="cuda")
        out = buf[1:S + 1, 8:8 + N]
        got = call_grouped(ops, a, w, sa, sw, off, rows=rows, bias=b, gelu=gelu, out=out)
        ops.check_status()
        want, slack, written = grouped64(a, w, off, rows, b, gelu, S, sa, sw)
        near(got[written], want[written], slack[written])
        assert (got[~written] == 7.0).all()              # rows behind the last expert's
        buf[1:S + 1, 8:8 + N] = 7.0
        assert (buf == 7.0).all()                        # and nothing around


@pytest.mark.parametrize("t", [BF16, torch.int8])
@pytest.mark.parametrize("S,N,K", [(6, 136, 64), (200, 136, 64), (2400, 136, 1024), (16400, 2568, 1024)])
def test_gemm_grouped_bad_indexes(ops, S, N, K, t):
    """Indexes outside A are rows of zeros; offsets outside the buffer or falling back reach nothing outside.  (Warp dot
    products, rows gathered in the kernel, and put in order first for CTA pairs.)"""
    g = gen(S)
    a, w, sa, sw = operands(g, t, 50, 4, N, K)
    rows = torch.randint(0, 50, (S,), generator=g, device="cuda", dtype=torch.int32)
    rows[1], rows[3], rows[4] = -1, 50, 2 ** 31 - 1
    bias = rand(g, 4, N)
    off = torch.tensor([0, 2, 2, 5, S], dtype=torch.int32, device="cuda")
    got = call_grouped(ops, a, w, sa, sw, off, rows=rows, bias=bias)
    want, slack, written = grouped64(a, w, off, rows, bias, False, S, sa, sw)
    near(got, want, slack)
    wild = torch.tensor([-5, 4, 1, 2 ** 31 - 1, 3], dtype=torch.int32, device="cuda")    # = 0..4, -, 4..S, -
    tame = torch.tensor([0, 4, 4, S, S], dtype=torch.int32, device="cuda")
    assert torch.equal(call_grouped(ops, a, w, sa, sw, wild, rows=rows, bias=bias),
                       call_grouped(ops, a, w, sa, sw, tame, rows=rows, bias=bias))
    ops.check_status()


@pytest.mark.parametrize("t", [BF16, torch.int8])
def test_gemm_grouped_without_scratch_and_with_an_odd_bias(ops, t):
    """A product large enough for CTA pairs whose caller has no scratch, or whose bias starts at an odd place."""
    from segment_anything_fast_b200 import _lib
    g = gen(12)
    S, M, E, N, K = 17000, 700, 3, 2568, 1024
    a, w, sa, sw = operands(g, t, M, E, N, K)
    rows = torch.randint(0, M, (S,), generator=g, device="cuda", dtype=torch.int32)
    off = torch.tensor([0, 4000, 12000, 16990], dtype=torch.int32, device="cuda")
    bias = rand(g, E * N + 1)[1:].reshape(E, N)
    want, slack, written = grouped64(a, w, off, rows, bias, True, S, sa, sw)
    got = call_grouped(ops, a, w, sa, sw, off, rows=rows, bias=bias, gelu=True)
    near(got[written], want[written], slack[written])
    lib, st, out = _lib.load(), ops.status_word(a.device), torch.full((S, N), 7.0, dtype=BF16, device="cuda")
    tail = (_lib.EPI_BIAS | _lib.EPI_GELU, None, st.data_ptr(), torch.cuda.current_stream().cuda_stream)
    bias = bias.clone()
    if t == torch.int8:
        rc = lib.samb_gemm_i8_grouped(a.data_ptr(), K, M, sa.data_ptr(), rows.data_ptr(), w.data_ptr(), K, N * K, sw.data_ptr(),
                                      bias.data_ptr(), off.data_ptr(), out.data_ptr(), N, S, E, N, K, *tail)
    else:
        rc = lib.samb_gemm_grouped(a.data_ptr(), K, M, rows.data_ptr(), w.data_ptr(), K, N * K, bias.data_ptr(), off.data_ptr(),
                                   out.data_ptr(), N, S, E, N, K, 0, *tail)
    assert rc == 0
    near(out[written], want[written], slack[written])
    assert (out[~written] == 7.0).all()
    ops.check_status()


@pytest.mark.parametrize("t", [BF16, torch.int8])
@pytest.mark.parametrize("S,N", [(6, 264), (700, 264), (20000, 2568)])
def test_gemm_grouped_captured_and_on_two_streams(ops, S, N, t):
    """Each kernel (warp dot products, single CTAs with gathered rows, ordered rows on CTA pairs) in two graphs replayed in
    turn over changing inputs, and in calls that overlap on two streams."""
    g = gen(S)
    E, K, M = 3, 512, 900
    a, w, sa, sw = operands(g, t, M, E, N, K)
    alt = [torch.flip(a, (0,)).contiguous(), a]
    rows = [torch.randint(0, M, (S,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    off = [torch.tensor([0, S // 5, S // 2, S], dtype=torch.int32, device="cuda"), torch.tensor([0, 0, S - 1, S], dtype=torch.int32, device="cuda")]
    bias = rand(g, E, N)
    call = lambda x, i: call_grouped(ops, x, w, sa, sw, off[i], rows=rows[i], bias=bias, gelu=True)
    want = [[call(x, i) for i in range(2)] for x in alt]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(alt[0], i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[0][i]) for o in got[i])
    del got
    x = alt[0].clone()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(call(x, i))
    for j in (1, 0, 1):
        x.copy_(alt[j])
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[j][i])
    ops.check_status()


@pytest.mark.parametrize("S", [4, 300])
def test_gemm_grouped_tells_rows_and_columns_apart(ops, S):
    """One-hot operands: every output says which row, column and expert it came from."""
    E, N, K = 3, 72, 64
    a = torch.zeros(S, K, dtype=BF16, device="cuda")
    a[torch.arange(S), torch.arange(S) % K] = 1.0
    w = (torch.arange(E, device="cuda")[:, None, None] * 64 + (torch.arange(N, device="cuda")[:, None] * 5 + torch.arange(K, device="cuda")) % 64).to(BF16)
    off = torch.tensor([0, S // 3, S // 3, S], dtype=torch.int32, device="cuda")
    got = ops.gemm_grouped(a, w, off)
    e = torch.where(torch.arange(S, device="cuda") < S // 3, 0, 2)
    want = w[e, :, torch.arange(S, device="cuda") % K]
    assert torch.equal(got, want)


def test_gemm_grouped_infinities_stay_in_their_rows(ops):
    for S in (5, 150):
        g = gen(S)
        a, w, _, _ = operands(g, BF16, S, 2, 64, 64)
        off = torch.tensor([0, 2, S], dtype=torch.int32, device="cuda")
        clean = ops.gemm_grouped(a, w, off)
        a[1, 3], a[3, 5] = math.inf, math.nan
        got = ops.gemm_grouped(a, w, off)
        keep = torch.ones(S, dtype=torch.bool, device="cuda")
        keep[[1, 3]] = False
        assert torch.equal(got[keep], clean[keep]) and not got[[1, 3]].isfinite().any()


# ------------------------------------------------------------------------------------------------ combination
@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("T,k,C", [(1, 1, 8), (1, 2, 1280), (33, 2, 1280), (1000, 3, 264), (517, 8, 64), (3, 5, 5120), (2000, 4, 768)])
def test_combine(ops, T, k, C, t):
    g = gen(T + k + C)
    x, r = rand(g, T * k + 3, C, t=t), rand(g, T, C, t=t)
    slots = torch.randperm(T * k, generator=g, device="cuda").int().reshape(T, k)
    slots[torch.rand(T, k, generator=g, device="cuda") < 0.2] = -1
    slots[0, 0] = T * k + 3                              # outside: nothing
    slots[-1] = -1                                       # a token that chose nobody
    w = rand(g, T, k)
    w[slots < 0] = math.nan                              # weights of no choice are not read
    ok = (slots >= 0) & (slots < x.shape[0])
    terms = torch.where(ok[..., None], x.double()[slots.long().clamp(0, x.shape[0] - 1)] * w.double().nan_to_num()[..., None], 0.0)
    for res in (r, None):
        got = ops.combine_topk(x, slots, w, residual=res)
        want = terms.sum(1) + (res.double() if res is not None else 0.0)
        near(got, want, (k + 1) * U32 * (terms.abs().sum(1) + (res.double().abs() if res is not None else 0.0)))
    wide = torch.zeros(T, C + 16, dtype=t, device="cuda")
    wide[:, 8:-8] = r
    ops.combine_topk(x, slots, w, residual=wide[:, 8:-8], out=wide[:, 8:-8])
    assert torch.equal(wide[:, 8:-8], ops.combine_topk(x, slots, w, residual=r)) and (wide[:, :8] == 0).all() and (wide[:, -8:] == 0).all()


# ------------------------------------------------------------------------------------------------ refusals on the device side
def test_wrapper_refusals(ops):
    h = torch.zeros(6, 64, dtype=BF16, device="cuda")
    f, f6 = torch.ones(64, device="cuda"), torch.ones(6, 2, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    fr = torch.ones(32, dtype=torch.float64, device="cuda")
    w = torch.zeros(2, 32, 64, dtype=BF16, device="cuda")
    w8, h8 = w.to(torch.int8), h.to(torch.int8)
    bad = [
        lambda: ops.block_norm(h.float()), lambda: ops.block_norm(h, h.half()), lambda: ops.block_norm(h, h[:5]),
        lambda: ops.block_norm(h, post=(f[:32], None)), lambda: ops.block_norm(h, pre=(f.bfloat16(), None)),
        lambda: ops.block_norm(h, gate=torch.ones(4, 64, device="cuda")), lambda: ops.block_norm(h.t()),
        lambda: ops.block_norm(h[:, :60]), lambda: ops.block_norm(h, out=h[:, :32]), lambda: ops.block_norm(h[0]),
        lambda: ops.block_norm(h[:, 1:57]), lambda: ops.block_norm_quant_i8(h.half(), None, None, (f, None)),
        lambda: ops.block_norm_quant_i8(h, None, None, None),
        lambda: ops.rotary(h, i32(0), fr), lambda: ops.rotary(h[None], i32(0, 1, 2, 3), fr), lambda: ops.rotary(h[None], f[:6], fr),
        lambda: ops.rotary(h[None], i32(0), fr.float()), lambda: ops.rotary(h[None], i32(0), torch.ones(33, dtype=torch.float64, device="cuda")),
        lambda: ops.rotary(h[None], torch.zeros(6, 3, dtype=torch.int32, device="cuda"), fr),
        lambda: ops.rotary(h[None].expand(3, 6, 64), i32(0), fr, out=h[None].expand(3, 6, 64)),
        lambda: ops.rotary(torch.zeros(1, 6, 12, dtype=BF16, device="cuda"), i32(0), fr[:4]),
        lambda: ops.route_topk(h, 2), lambda: ops.route_topk(f6, 3), lambda: ops.route_topk(f6, 0),
        lambda: ops.route_topk(f6, 1, bias=f), lambda: ops.route_topk(f6.t(), 1), lambda: ops.route_topk(torch.zeros(2, 513, device="cuda"), 1),
        lambda: ops.gemm_grouped(h, w.half(), i32(0, 3, 6)), lambda: ops.gemm_grouped(h, w, i32(0, 6)),
        lambda: ops.gemm_grouped(h, w, i32(0, 3, 6).long()), lambda: ops.gemm_grouped(h[:, :32], w, i32(0, 3, 6)),
        lambda: ops.gemm_grouped(h, w, i32(0, 3, 6), bias=f), lambda: ops.gemm_grouped(h, w, i32(0, 3, 6), rows=i32(0, 1).long()),
        lambda: ops.gemm_grouped(h, w, i32(0, 3, 6), out=h), lambda: ops.gemm_grouped(h8, w8, i32(0, 3, 6)),
        lambda: ops.gemm_grouped(h, w.transpose(1, 2), i32(0, 3, 6)),
        lambda: ops.gemm_i8_grouped(h8, f[:5], w8, torch.ones(2, 32, device="cuda"), i32(0, 3, 6)),
        lambda: ops.gemm_i8_grouped(h8, None, w8, torch.ones(2, 32, device="cuda"), i32(0, 3, 6)),
        lambda: ops.combine_topk(h, i32(0, 1), f6), lambda: ops.combine_topk(h, i32(0, 1, 2, 3).reshape(2, 2), f6),
        lambda: ops.combine_topk(h, i32(0, 1, 2, 3).reshape(2, 2), f6[:2], residual=h[:3]),
        lambda: ops.combine_topk(h, torch.zeros(6, 9, dtype=torch.int32, device="cuda"), torch.ones(6, 9, device="cuda")),
        lambda: ops.combine_topk(h, torch.zeros(6, 2, dtype=torch.int32, device="cuda"), f6, out=h),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {n} was not refused")


def test_tensors_of_another_device_are_refused(ops, monkeypatch):
    h, f = torch.zeros(8, 64, dtype=BF16, device="cuda"), torch.ones(64, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    w = torch.zeros(2, 32, 64, dtype=BF16, device="cuda")
    w8, h8, f8, f2 = w.to(torch.int8), h.to(torch.int8), torch.ones(8, device="cuda"), torch.ones(2, 32, device="cuda")
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    for call in (lambda: ops.block_norm(h), lambda: ops.block_norm_quant_i8(h, None, None, (f, None)),
                 lambda: ops.rotary(h[None], i[:1], torch.ones(32, dtype=torch.float64, device="cuda")),
                 lambda: ops.route_topk(f.reshape(8, 8), 2), lambda: ops.gemm_grouped(h, w, i),
                 lambda: ops.gemm_i8_grouped(h8, f8, w8, f2, i), lambda: ops.combine_topk(h, i[:2].reshape(1, 2), f[:2].reshape(1, 2))):
        with pytest.raises(RuntimeError, match="current device is cuda:1"):
            call()


def test_first_call_inside_a_capture_is_refused(ops, monkeypatch):
    """The status word of a device outlives every graph: a capture may not be what allocates it."""
    h, w = torch.zeros(8, 64, dtype=BF16, device="cuda"), torch.zeros(2, 32, 64, dtype=BF16, device="cuda")
    i = torch.zeros(3, dtype=torch.int32, device="cuda")
    monkeypatch.setattr(ops, "_status_words", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        ops.gemm_grouped(h, w, i)


def test_offsets_past_32_bits(ops):
    """Tensors of more than 2^31 elements: the last rows are as right as the first."""
    g = gen(2)
    rows, C = (1 << 31) // 1280 + 7001, 1280
    pick = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device="cuda")
    x = torch.empty(rows, C, dtype=BF16, device="cuda")
    for lo in range(0, rows, 1 << 18):                   # rows of few different values, made in pieces
        x[lo:lo + (1 << 18)] = (torch.arange(lo, min(rows, lo + (1 << 18)), device="cuda")[:, None] * 7 + torch.arange(C, device="cuda") * 3).remainder(251).to(BF16) / 64
    pre = (rand(g, C), rand(g, C))
    few = x[pick].contiguous()
    a, y = ops.block_norm(x, x, post=pre, pre=pre)
    wa, wy = ops.block_norm(few, few, post=pre, pre=pre)
    x64, ex, y64, ey = block64(few, few, pre, pre, None, 1.0, False)
    near(a[pick], x64, ex)
    near(y[pick], y64, ey)
    near(wa, x64, ex)
    del a, y
    # one plane of heads of 64, then of positions: rows past 2^31 / 64
    planes = x.view(-1)[: 2 * ((1 << 30) // 64 + 64) * 64].view(2, -1, 64)
    freqs, _ = ops.rotary_freqs(64)
    pos = torch.arange(64, device="cuda")
    out = ops.rotary(planes, pos, freqs)
    assert torch.equal(out[1, -64:], ops.rotary(planes[1:, -64:].contiguous(), pos, freqs)[0])
    assert torch.equal(out[0, :64], ops.rotary(planes[:1, :64].contiguous(), pos, freqs)[0])
    del out, planes
    # combination and grouped products: the last tokens choose the last rows
    T = rows // 2
    slots = torch.arange(2 * T, device="cuda", dtype=torch.int32).reshape(T, 2)
    wts = torch.rand(T, 2, generator=g, device="cuda")
    out = ops.combine_topk(x, slots, wts)
    end = torch.tensor([T - 2, T - 1], device="cuda")
    terms = x[slots[end].long()].double() * wts[end].double()[..., None]
    near(out[end], terms.sum(1), 3 * U32 * terms.abs().sum(1))
    del out
    w = rand(g, 3, C, 64, by=0.1, t=BF16)
    off = torch.tensor([0, 5, rows - 300, rows], dtype=torch.int32, device="cuda")
    tall = x[:, :64]                                     # leading dimension 1280: A reaches past 2^31 elements too
    src = torch.arange(rows - 1, -1, -1, device="cuda", dtype=torch.int32)
    for idx in (None, src):
        out = ops.gemm_grouped(tall, w, off, rows=idx)
        ops.check_status()
        e = torch.tensor([0, 1, 1, 2, 2], device="cuda")
        at = torch.tensor([4, 5, rows // 2, rows - 300, rows - 1], device="cuda")
        ar = tall[at if idx is None else src[at].long()].double()
        want = torch.einsum("sk,snk->sn", ar, w[e].double())
        near(out[at], want, 64 * 2.0 ** -23 * torch.einsum("sk,snk->sn", ar.abs(), w[e].double().abs()))
        del out


def test_empty_calls(ops):
    z = torch.zeros(0, 64, dtype=BF16, device="cuda")
    f = torch.ones(64, device="cuda")
    x, y = ops.block_norm(z, z, pre=(f, f))
    assert x.shape == y.shape == (0, 64)
    fr = torch.ones(32, dtype=torch.float64, device="cuda")
    assert ops.rotary(z[None], torch.zeros(5, dtype=torch.int32, device="cuda"), fr).shape == (1, 0, 64)
    w = torch.zeros(2, 32, 64, dtype=BF16, device="cuda")
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.gemm_grouped(z, w, off).shape == (0, 32)
    assert ops.combine_topk(z, off[:0].reshape(0, 2), f[:0].reshape(0, 2)).shape == (0, 64)
    r = torch.ones(1, 64, dtype=BF16, device="cuda")      # nobody chose anything: the residual comes back
    assert torch.equal(ops.combine_topk(z, torch.full((1, 2), -1, dtype=torch.int32, device="cuda"), torch.zeros(1, 2, device="cuda"), r), r)


# ------------------------------------------------------------------------------------------------ together
class Block:
    """One transformer block on a 64 x 64 token raster: rotary attention, norms on both sides of each branch with an
    image's own gate, mixture of experts."""

    def __init__(self, ops, t=BF16, quant=False, B=2, C=160, H=2, E=5, k=2, hidden=320):
        g = gen(77)
        self.ops, self.B, self.C, self.H, self.k, self.quant = ops, B, C, H, k, quant
        lin = lambda n, m, *e: rand(g, *e, n, m, by=1 / math.sqrt(m), t=BF16)
        self.wqkv, self.bqkv, self.wo = lin(3 * C, C), rand(g, 3 * C), lin(C, C)
        self.norms = [(rand(g, C, by=0.1, at=1.0), rand(g, C, by=0.1)) for _ in range(5)]
        self.gates = [rand(g, B, C, by=0.2, at=0.5) for _ in range(2)]
        self.router = lin(8 * ((E + 7) // 8), C)          # the GEMM's rows come in eights; the router sees E of them
        self.E, self.w1, self.b1, self.w2 = E, lin(hidden, C, E), rand(g, E, hidden), lin(C, hidden, E)
        if quant:
            def q(w):
                s = w.float().abs().amax(2) / 127
                return torch.round(w.float() / s[..., None]).clamp(-127, 127).to(torch.int8), s
            (self.w1q, self.s1), (self.w2q, self.s2) = q(self.w1), q(self.w2)
        p = torch.arange(4096, device="cuda")
        self.pos = torch.stack([p % 64, p // 64], 1)
        self.freqs, _ = ops.rotary_freqs(C // H, axes=2)
        self.tables = torch.zeros(256, C // H, dtype=BF16, device="cuda")

    def __call__(self, x, y, see=None):
        """Stream x and its normed form y -> the same after the block."""
        o, C, H, d = self.ops, self.C, self.H, self.C // self.H
        see = see if see is not None else {}
        qkv = o.gemm_heads(y, None, self.wqkv, None, self.bqkv, d)
        see["qkv"] = qkv.clone()
        o.rotary(qkv[:2 * H], self.pos, self.freqs, out=qkv[:2 * H])
        a = o.gemm_bf16(o.attn_relpos_global_tables(qkv, self.tables, self.B, H, 4096, d), self.wo)
        x1, y1 = o.block_norm(a, x, post=self.norms[0], pre=self.norms[1], gate=self.gates[0])
        logits = o.gemm_bf16(y1, self.router, raw=True)[:, :self.E]
        r = o.route_topk(logits, self.k)
        if self.quant:
            yq, ys = o.quant_rows_i8(y1)
            hid = o.gemm_i8_grouped(yq, ys, self.w1q, self.s1, r.offsets, rows=r.rows, bias=self.b1, gelu=True)
            hq, hs = o.quant_rows_i8(hid)
            back = o.gemm_i8_grouped(hq, hs, self.w2q, self.s2, r.offsets)
        else:
            hid = o.gemm_grouped(y1, self.w1, r.offsets, rows=r.rows, bias=self.b1, gelu=True)
            back = o.gemm_grouped(hid, self.w2, r.offsets)
        m = o.combine_topk(back, r.slots, r.weights)
        see.update(rot=qkv, a=a, x=x, x1=x1, y1=y1, logits=logits, r=r, hid=hid, back=back, m=m)
        return o.block_norm(m, x1, post=self.norms[2], pre=self.norms[3], gate=self.gates[1])


def test_block_together(ops):
    b = Block(ops)
    g = gen(78)
    x = rand(g, b.B * 4096, b.C, t=BF16)
    y = ops.layernorm(x, *b.norms[4])
    see = {}
    x2, y2 = b(x, y, see)
    ops.check_status()
    planes = 2 * b.H
    want, slack = rotary64(see["qkv"][:planes], b.pos, b.freqs, False, 1.0)
    near(see["rot"][:planes], want, slack)
    assert torch.equal(see["rot"][planes:], see["qkv"][planes:])
    x64, ex, y64, ey = block64(see["a"], x, b.norms[0], b.norms[1], b.gates[0], 1.0, False)
    near(see["x1"], x64, ex)
    near(see["y1"], y64, ey)
    r = check_route(ops, see["logits"], b.k)
    for p, q in zip(r, see["r"]):
        assert torch.equal(p, q)
    S = r.rows.numel()
    h64, eh, _ = grouped64(see["y1"], b.w1, r.offsets, r.rows, b.b1, True, S)
    near(see["hid"], h64, eh)
    k64, ek, _ = grouped64(see["hid"], b.w2, r.offsets, None, None, False, S)
    near(see["back"], k64, ek)
    terms = see["back"].double()[r.slots.long()] * r.weights.double()[..., None]
    near(see["m"], terms.sum(1), (b.k + 1) * U32 * terms.abs().sum(1))
    x64, ex, y64, ey = block64(see["m"], see["x1"], b.norms[2], b.norms[3], b.gates[1], 1.0, False)
    near(x2, x64, ex)
    near(y2, y64, ey)


def test_block_int8_near_bf16(ops):
    """The int8 experts against the bf16 ones, row by row: two products with operands rounded to a 254th of their
    largest value.  Rounding is worth at most (1/254) |a|max |w|max K^(1/2) ~ 2 % of the result's size in the mean."""
    x = rand(gen(78), 2 * 4096, 160, t=BF16)
    one, two = Block(ops), Block(ops, quant=True)
    y = ops.layernorm(x, *one.norms[4])
    s1, s2 = {}, {}
    one(x, y, s1)
    two(x, y, s2)
    assert torch.equal(s1["r"].ids, s2["r"].ids)
    rel = (s1["m"].double() - s2["m"].double()).norm() / s1["m"].double().norm()
    assert rel < 0.03


@pytest.mark.parametrize("quant", [False, True])
def test_block_captured_on_another_stream(ops, quant):
    """Two captured graphs of the same block replayed in turn, and eager calls on two streams at once, all give the
    eager call's bits."""
    b = Block(ops, quant=quant)
    xs = [rand(gen(80 + i), b.B * 4096, b.C, t=BF16) for i in range(2)]
    ys = [ops.layernorm(x, *b.norms[4]) for x in xs]
    want = [b(x, y) for x, y in zip(xs, ys)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(b(xs[i], ys[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o[0], want[i][0]) and torch.equal(o[1], want[i][1])
    graphs, outs, ins = [], [], []
    for i in range(2):
        gr, x, y = torch.cuda.CUDAGraph(), xs[i].clone(), ys[i].clone()
        with torch.cuda.graph(gr):
            outs.append(b(x, y))
        graphs.append(gr)
        ins.append((x, y))
    for turn in range(2):
        for i in range(2):
            j = (i + turn) % 2                            # other inputs in the same buffers
            ins[i][0].copy_(xs[j])
            ins[i][1].copy_(ys[j])
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            j = (i + turn) % 2
            assert torch.equal(outs[i][0], want[j][0]) and torch.equal(outs[i][1], want[j][1])
    ops.check_status()

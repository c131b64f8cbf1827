"""Measured cases of the transformer-block operators beside the encoder's own: the norms around a block, rotary
positions, and a mixture of experts (router, products grouped by expert, combination of the chosen experts).

``run`` computes an operator in its plain form (elementary torch operations) or, with ``own``, through the package.
The sizes are those of the encoder (64 x 64 tokens an image, width 1280, 16 heads of 80, MLP width 5120) from a single
token up to a batch of images, and smaller and odd ones around them.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one token through the norms between two blocks: what a step-by-step caller pays, all latency
        {"name": "norm, one token", "op": "norm", "rows": 1, "width": 1280, "images": 1, "type": "bf16", "rms": False,
         "post": True},
        # the residual stream of a batch of 32 images with a gate vector an image
        {"name": "norm, 32 images", "op": "norm", "rows": 32 * 4096, "width": 1280, "images": 32, "type": "bf16",
         "rms": False, "post": True},
        # the queries and keys of one token far into a stretched context
        {"name": "rotary, one token", "op": "rotary", "planes": 32, "rows": 1, "dim": 80, "rot": 64, "axes": 1,
         "interleaved": True, "type": "f16", "period": 1, "far": 1000000, "factor": 8.0},
        # the query and key planes of 8 images, column and row of the raster as the two coordinates
        {"name": "rotary, 8 images", "op": "rotary", "planes": 32, "rows": 8 * 4096, "dim": 80, "rot": 80, "axes": 2,
         "interleaved": False, "type": "bf16", "period": 4096, "far": 64, "factor": 1.0},
        # the router's choice for one token
        {"name": "route, one token", "op": "route", "tokens": 1, "experts": 16, "k": 2, "sigmoid": False, "bias": False},
        # the router's choice for 8 images, with a balancing bias and padded tokens
        {"name": "route, 8 images", "op": "route", "tokens": 8 * 4096, "experts": 64, "k": 4, "sigmoid": True,
         "bias": True},
        # first MLP product of the chosen experts: one token
        {"name": "experts, one token", "op": "experts", "tokens": 1, "experts": 16, "k": 2, "n": 5120, "kdim": 1280,
         "type": "bf16", "gather": True, "gelu": True, "bias": True},
        # second MLP product for a ragged handful of tokens, rows already in the experts' order
        {"name": "experts, 1031 tokens back", "op": "experts", "tokens": 1031, "experts": 16, "k": 2, "n": 1280,
         "kdim": 5120, "type": "f16", "gather": False, "gelu": False, "bias": True},
        # first MLP product for 8 images
        {"name": "experts, 8 images", "op": "experts", "tokens": 8 * 4096, "experts": 16, "k": 2, "n": 5120,
         "kdim": 1280, "type": "bf16", "gather": True, "gelu": True, "bias": True},
        # the same for 2 images in the int8 mode
        {"name": "experts, 2 images int8", "op": "experts", "tokens": 2 * 4096, "experts": 8, "k": 2, "n": 5120,
         "kdim": 1280, "type": "i8", "gather": True, "gelu": True, "bias": True},
        # weighted sum of the chosen experts' rows: one token, then 8 images
        {"name": "combine, one token", "op": "combine", "tokens": 1, "experts": 16, "k": 2, "width": 1280,
         "type": "bf16", "residual": True},
        {"name": "combine, 8 images", "op": "combine", "tokens": 8 * 4096, "experts": 16, "k": 2, "width": 1280,
         "type": "bf16", "residual": True},
    ]


def _log(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))
    return max(lo, min(hi, v // step * step))


def draw(rng):
    op = rng.choice(["norm", "rotary", "route", "experts", "experts", "combine"])
    if op == "norm":
        images = rng.choice([1, 1, 2, 5, 8])
        return {"op": op, "rows": images * _log(rng, 1, 16384), "width": _log(rng, 64, 1280, 8), "images": images,
                "type": rng.choice(["bf16", "f16"]), "rms": rng.random() < 0.5, "post": rng.random() < 0.7}
    if op == "rotary":
        dim = _log(rng, 16, 256, 8)
        axes = rng.choice([1, 2])
        rot = dim if rng.random() < 0.5 else max(4, dim // 2 // 4 * 4)
        period = _log(rng, 1, 4096)
        return {"op": op, "planes": rng.randint(1, 40), "rows": period * rng.randint(1, 4), "dim": dim, "rot": rot,
                "axes": axes, "interleaved": rng.random() < 0.5, "type": rng.choice(["bf16", "f16"]), "period": period,
                "far": _log(rng, 64, 1000000), "factor": rng.choice([1.0, 2.0, 8.0])}
    if op == "route":
        e = _log(rng, 2, 256)
        return {"op": op, "tokens": _log(rng, 1, 32768), "experts": e, "k": rng.randint(1, min(8, e)),
                "sigmoid": rng.random() < 0.5, "bias": rng.random() < 0.5}
    tokens, k = _log(rng, 1, 16384), rng.randint(1, 4)
    if op == "combine":
        return {"op": op, "tokens": tokens, "experts": _log(rng, 4, 64), "k": k, "width": _log(rng, 64, 1280, 8),
                "type": rng.choice(["bf16", "f16"]), "residual": rng.random() < 0.5}
    return {"op": op, "tokens": tokens, "experts": _log(rng, 4, 32), "k": k, "n": _log(rng, 64, 5120, 8),
            "kdim": _log(rng, 64, 1280, 16), "type": rng.choice(["bf16", "f16", "i8"]), "gather": rng.random() < 0.5,
            "gelu": rng.random() < 0.5, "bias": rng.random() < 0.7}


# ---------------------------------------------------------------------------------------------------- inputs
def _freqs(c, dev):
    """Angular frequencies of the pairs (radians a position) and the factor on the rotation.  With ``factor`` > 1 the
    slow pairs are stretched by it, the fast ones kept, with a ramp between 1 and 32 turns over 4096 positions."""
    n = c["rot"] // 2 // c["axes"]
    i = torch.arange(n, dtype=torch.float64, device=dev)
    f = 10000.0 ** (-i / n)
    mscale = 1.0
    if c["factor"] > 1:
        turns = 4096.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        f = f * (keep + (1 - keep) / c["factor"])
        mscale = 0.1 * math.log(c["factor"]) + 1.0
    return torch.cat([f] * c["axes"]) if c["axes"] > 1 else f, mscale


def _plan(c, g, dev):
    """A skewed choice of k different experts a token, and the order of the chosen rows by expert."""
    T, E, k = c["tokens"], c["experts"], min(c["k"], c["experts"])
    score = torch.randn(T, E, generator=g, device=dev) + 0.7 * torch.randn(E, generator=g, device=dev)
    ids = score.topk(k, dim=1).indices
    order = torch.sort(ids.reshape(-1), stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=dev)
    counts = torch.bincount(ids.reshape(-1), minlength=E)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    w = torch.rand(T, k, generator=g, device=dev) + 0.1
    w = w / w.sum(1, keepdim=True)
    return ((order // k).to(torch.int32), slots.reshape(T, k).to(torch.int32), offsets.to(torch.int32), w,
            int(counts.max()))


def prepare(case, seed):
    c, dev = dict(case), torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape, by=1.0):
        return torch.randn(*shape, generator=g, device=dev) * by

    s = {"case": c}
    if c["op"] == "norm":
        t, n = _TYPES[c["type"]], c["width"]
        # a stream with a few strong channels, as residual streams have
        strong = 1 + 10 * (torch.rand(n, generator=g, device=dev) < 0.01)
        s["h"] = (rand(c["rows"], n) * strong + 0.1).to(t)
        s["residual"] = (rand(c["rows"], n, by=2.0) * strong - 0.2).to(t)
        s["post"] = (1 + rand(n, by=0.1), None if c["rms"] else rand(n, by=0.1)) if c["post"] else None
        s["pre"] = (1 + rand(n, by=0.1), None if c["rms"] else rand(n, by=0.1))
        s["gate"] = 0.5 + rand(c["images"], n, by=0.2)
        s["scale"] = 0.9
    elif c["op"] == "rotary":
        s["x"] = rand(c["planes"], c["rows"], c["dim"]).to(_TYPES[c["type"]])
        if c["axes"] == 2:
            p = torch.arange(c["period"], device=dev)
            s["positions"] = torch.stack([p % c["far"], p // c["far"] + seed % 7], dim=1)
        else:
            s["positions"] = torch.randint(0, c["far"] + 1, (c["period"],), generator=g, device=dev)
        s["freqs"], s["mscale"] = _freqs(c, dev)
    elif c["op"] == "route":
        T, E = c["tokens"], c["experts"]
        x = rand(T, E) + rand(E, by=0.5)
        x = x.to(torch.bfloat16).float()                 # a router in bf16: ties are common
        x[torch.rand(T, E, generator=g, device=dev) < 0.02] = -math.inf       # experts switched off for a token
        x[T - T // 50:] = -math.inf                      # padded tokens choose nobody
        s["logits"] = x
        s["bias"] = rand(E, by=0.1) if c["bias"] else None
    elif c["op"] == "experts":
        rows, _, offsets, _, s["most"] = _plan(c, g, dev)
        s["offsets"], s["rows"] = offsets, rows if c["gather"] else None
        m = c["tokens"] if c["gather"] else rows.numel()
        E, n, k = c["experts"], c["n"], c["kdim"]
        s["bias"] = rand(E, n, by=0.5) if c["bias"] else None
        if c["type"] == "i8":
            s["a"] = torch.randint(-127, 128, (m, k), generator=g, device=dev, dtype=torch.int8)
            s["w"] = torch.randint(-127, 128, (E, n, k), generator=g, device=dev, dtype=torch.int8)
            s["a_scale"] = (0.5 + torch.rand(m, generator=g, device=dev)) / 50
            s["w_scale"] = (0.5 + torch.rand(E, n, generator=g, device=dev)) / (60 * math.sqrt(k))
        else:
            s["a"] = rand(m, k).to(_TYPES[c["type"]])
            s["w"] = rand(E, n, k, by=1 / math.sqrt(k)).to(_TYPES[c["type"]])
    else:
        rows, s["slots"], _, s["weights"], _ = _plan(c, g, dev)
        s["x"] = rand(rows.numel(), c["width"]).to(_TYPES[c["type"]])
        s["residual"] = rand(c["tokens"], c["width"]).to(_TYPES[c["type"]]) if c["residual"] else None
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_norm(x, affine, rms):
    if rms:
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
    else:
        x = x - x.mean(1, keepdim=True)
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + 1e-6)
    x = x * affine[0]
    return x if affine[1] is None else x + affine[1]


def _plain(s):
    c = s["case"]
    if c["op"] == "norm":
        t = s["h"].dtype
        u = s["h"].float()
        if s["post"] is not None:
            u = _plain_norm(u, s["post"], c["rms"])
        u = (u.reshape(c["images"], -1, c["width"]) * s["gate"][:, None, :]).reshape(c["rows"], c["width"])
        x = s["scale"] * s["residual"].float() + u
        return x.to(t), _plain_norm(x, s["pre"], c["rms"]).to(t)
    if c["op"] == "rotary":
        n, half = c["rot"], c["rot"] // 2
        p = s["positions"].reshape(c["period"], c["axes"]).double()
        angle = p.repeat_interleave(half // c["axes"], dim=1) * s["freqs"]
        again = c["rows"] // c["period"]
        cos, sin = ((f(angle) * s["mscale"]).float().repeat(again, 1) for f in (torch.cos, torch.sin))
        x = s["x"].float()
        if c["interleaved"]:
            a, b = x[..., 0:n:2], x[..., 1:n:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(2)
        else:
            a, b = x[..., :half], x[..., half:n]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([r, x[..., n:]], dim=-1).to(s["x"].dtype)
    if c["op"] == "route":
        x, k, (T, E) = s["logits"], c["k"], s["logits"].shape
        key = x if s["bias"] is None else x + s["bias"]
        top, ids = torch.sort(key, dim=1, descending=True, stable=True)
        none = top[:, :k] == -math.inf
        ids = ids[:, :k]
        if c["sigmoid"]:
            p = 1 / (1 + torch.exp(-x))
        else:
            m = x.amax(1, keepdim=True)
            p = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
            p = p / p.sum(1, keepdim=True)
        w = torch.where(none, torch.zeros_like(top[:, :k]), p.gather(1, ids))
        total = w.sum(1, keepdim=True)
        w = torch.where(total > 0, w / total, torch.zeros_like(w))
        ids = torch.where(none, torch.full_like(ids, -1), ids)
        flat = torch.where(ids < 0, torch.full_like(ids, E), ids).reshape(-1)
        by, order = torch.sort(flat, stable=True)
        offsets = torch.searchsorted(by, torch.arange(E + 1, device=x.device))
        at = torch.arange(T * k, device=x.device)
        slots = torch.empty_like(order)
        slots[order] = torch.where(by < E, at, torch.full_like(at, -1))
        rows = torch.where(by < E, order // k, torch.full_like(order, -1))
        return tuple(v.to(torch.int32) for v in (ids, slots.reshape(T, k), rows, offsets)) + (w,)
    if c["op"] == "experts":
        o, S = s["offsets"].long(), s["rows"].numel() if c["gather"] else s["a"].shape[0]
        place = (o[:-1, None] + torch.arange(s["most"], device=o.device)).clamp(max=S - 1)      # [E, most]
        src = s["rows"].long()[place] if c["gather"] else place
        slot = torch.arange(S, device=o.device)
        expert = torch.searchsorted(o, slot, right=True) - 1
        if c["type"] == "i8":                            # long sums of whole numbers: 64 bits keep them whole
            y = torch.bmm(s["a"].double()[src], s["w"].double().transpose(1, 2)).float()
            y = y * s["a_scale"][src][..., None] * s["w_scale"][:, None, :]
        else:
            y = torch.bmm(s["a"].float()[src], s["w"].float().transpose(1, 2))
        if s["bias"] is not None:
            y = y + s["bias"][:, None, :]
        if c["gelu"]:
            y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
        return y[expert, slot - o[expert]].to(torch.bfloat16 if c["type"] == "i8" else s["a"].dtype)
    y = (s["x"].float()[s["slots"].long()] * s["weights"][..., None]).sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------------------------------- the package's
def _own(s):
    from segment_anything_fast_b200 import ops
    c = s["case"]
    if c["op"] == "norm":
        return ops.block_norm(s["h"], s["residual"], post=s["post"], pre=s["pre"], gate=s["gate"],
                              res_scale=s["scale"], rms=c["rms"])
    if c["op"] == "rotary":
        return ops.rotary(s["x"], s["positions"], s["freqs"], interleaved=c["interleaved"], mscale=s["mscale"])
    if c["op"] == "route":
        r = ops.route_topk(s["logits"], c["k"], bias=s["bias"], sigmoid=c["sigmoid"])
        return r.ids, r.slots, r.rows, r.offsets, r.weights
    if c["op"] == "experts":
        if c["type"] == "i8":
            return ops.gemm_i8_grouped(s["a"], s["a_scale"], s["w"], s["w_scale"], s["offsets"], rows=s["rows"],
                                       bias=s["bias"], gelu=c["gelu"])
        return ops.gemm_grouped(s["a"], s["w"], s["offsets"], rows=s["rows"], bias=s["bias"], gelu=c["gelu"])
    return ops.combine_topk(s["x"], s["slots"], s["weights"], residual=s["residual"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------------------------------- work
def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        return {"bytes": 8 * n + 4 * c["width"] * (c["images"] + 4), "flops": 20 * n}
    if c["op"] == "rotary":
        n = c["planes"] * c["rows"] * c["dim"]
        return {"bytes": 4 * n + 8 * c["period"] * c["axes"], "flops": 3 * n}
    if c["op"] == "route":
        return {"bytes": 4 * c["tokens"] * (c["experts"] + 4 * c["k"]) + 4 * c["experts"],
                "flops": 4 * c["tokens"] * c["experts"]}
    S, e = c["tokens"] * min(c["k"], c["experts"]), 1 if c["type"] == "i8" else 2
    if c["op"] == "experts":
        m = c["tokens"] if c["gather"] else S
        used = min(c["experts"], S)
        return {"bytes": e * c["kdim"] * (m + used * c["n"]) + 2 * S * c["n"], "flops": 2 * S * c["n"] * c["kdim"]}
    return {"bytes": 2 * c["width"] * (S + c["tokens"] * (2 if c["residual"] else 1)) + 8 * S,
            "flops": 2 * S * c["width"]}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _norm64(v, affine, rms):
    centre = v if rms else v - v.sum(-1, keepdim=True) / v.shape[-1]
    v = centre / torch.sqrt((centre ** 2).sum(-1, keepdim=True) / v.shape[-1] + 1e-6) * affine[0].double()
    return v if affine[1] is None else v + affine[1].double()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "norm":
        each, xs, ys = c["rows"] // c["images"], [], []
        for i in range(c["images"]):
            h = s["h"][i * each:(i + 1) * each].double()
            if s["post"] is not None:
                h = _norm64(h, s["post"], c["rms"])
            xs.append(s["residual"][i * each:(i + 1) * each].double() * s["scale"] + h * s["gate"][i].double())
            ys.append(_norm64(xs[-1], s["pre"], c["rms"]))
        return torch.cat(xs), torch.cat(ys)
    if c["op"] == "rotary":
        half, each = c["rot"] // 2, c["rot"] // 2 // c["axes"]
        pos = s["positions"].reshape(c["period"], c["axes"])
        pos = pos[torch.arange(c["rows"], device=pos.device) % c["period"]].double()
        y = s["x"].double()
        for i in range(half):
            i0, i1 = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
            z = torch.polar(torch.full_like(pos[:, 0], s["mscale"]), pos[:, i // each] * s["freqs"][i])
            z = z * torch.complex(s["x"][..., i0].double(), s["x"][..., i1].double())
            y[..., i0], y[..., i1] = z.real, z.imag
        return y
    if c["op"] == "route":
        x = s["logits"].double()
        choice = s["logits"] if s["bias"] is None else s["logits"] + s["bias"]
        p = torch.sigmoid(x) if c["sigmoid"] else torch.softmax(x, 1).nan_to_num(0.0)
        w, left = [], choice.clone()
        for _ in range(c["k"]):                          # the largest, lowest index first, one after the other
            best = left.amax(1, keepdim=True)
            at = (left == best).to(torch.int8).argmax(1, keepdim=True)
            w.append(torch.where(best == -math.inf, torch.zeros_like(p[:, :1]), p.gather(1, at)))
            left.scatter_(1, at, -math.inf)
        w = torch.cat(w, 1)
        return None, None, None, None, (w / w.sum(1, keepdim=True)).nan_to_num(0.0)
    if c["op"] == "experts":
        S = s["rows"].numel() if c["gather"] else s["a"].shape[0]
        out = torch.empty(S, c["n"], dtype=torch.float64, device=s["a"].device)
        ends = s["offsets"].tolist()
        for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
            pick = s["rows"][lo:hi].long() if c["gather"] else slice(lo, hi)
            y = s["a"][pick].double() @ s["w"][e].double().t()
            if c["type"] == "i8":
                y = y * s["a_scale"][pick].double()[:, None] * s["w_scale"][e].double()
            if s["bias"] is not None:
                y = y + s["bias"][e].double()
            out[lo:hi] = y * torch.special.ndtr(y) if c["gelu"] else y
        return out
    y = torch.zeros(c["tokens"], c["width"], dtype=torch.float64, device=s["x"].device)
    if s["residual"] is not None:
        y += s["residual"].double()
    for j in range(s["slots"].shape[1]):
        y += s["x"][s["slots"][:, j].long()].double() * s["weights"][:, j:j + 1].double()
    return y

"""Workloads of the token operators (``wst_amd.tokens``): layer norm, rotary positions with several axes, and
attention with capped scores, a distance bias, documents or a prefix.

The sizes come from the scattering geometries of this repository: pooled features and coefficient maps of 64x64 RGB
(J=2: 243 x 16x16, J=4: 1251 x 4x4), of 128x128 RGB (J=2: 243 x 32x32) and of 256x256 with four bands
(J=6, L=12: 8932 x 4x4), as rows of features or as sequences of map positions, one patch or many packed together.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BASE = 10000.0
EPS = 1e-5
GRID = 16          # side of the token grid behind the positions: the 64x64, J=2 maps


# ------------------------------------------------------------------------------------------------ cases
def _norm(name, layout, lead, n, points, dtype, out, train, x_grad):
    c = {"op": "norm", "layout": layout, "lead": lead, "n": n, "points": points, "dtype": dtype, "out": out,
         "train": train, "x_grad": x_grad}
    return dict(c, name=name) if name else c


def _rotary(name, batch, tokens, heads, kv_heads, dim, time, rows, cols, interleaved, dtype, train):
    c = {"op": "rotary", "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "time": time, "rows": rows, "cols": cols, "interleaved": interleaved, "dtype": dtype, "train": train}
    return dict(c, name=name) if name else c


def _attention(name, batch, tq, tk, heads, kv_heads, dim, dtype, cap, bias, mask, documents, ragged, train):
    c = {"op": "attention", "batch": batch, "tq": tq, "tk": tk, "heads": heads, "kv_heads": kv_heads, "dim": dim,
         "dtype": dtype, "cap": cap, "bias": bias, "mask": mask, "documents": documents, "ragged": ragged,
         "train": train}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one classifier call on the pooled features of 64 patches (128x128 RGB, J=2: 486 a patch): latency
        _norm("norm pooled", "rows", 64, 486, 1, "f32", "f32", False, False),
        # maps of 1024 RGB patches of 64x64, J=4, read where the transform left them, tokens out for a bf16 network; the
        # transform has no gradient, so a training step needs the weight's and the bias's alone
        _norm("norm maps J=4 train", "maps", 1024, 1251, 16, "f32", "bf16", True, False),
        # maps of the 128x128 geometry for inference
        _norm("norm maps 128 J=2", "maps", 160, 243, 1024, "f32", "f32", False, False),
        # hidden tokens of a network behind the transform, whole training step
        _norm("norm tokens train", "rows", 32768, 1024, 1, "bf16", "bf16", True, True),
        # a read-out query and the newest token's key for each of 64 series: latency
        _rotary("rotary one token", 64, 1, 8, 2, 64, 8, 12, 12, False, "bf16", False),
        # a time series of sixteen 16x16 maps, training step
        _rotary("rotary series train", 4, 4096, 16, 4, 128, 16, 24, 24, False, "bf16", True),
        # single 32x32 maps in float32, part of a head of an odd width turned
        _rotary("rotary maps f32", 32, 1024, 4, 4, 40, 0, 7, 9, True, "f32", False),
        # a read-out query over a stored series of up to 4096 positions for each of 64 fields
        _attention("attention one query", 64, 1, 4096, 8, 2, 64, "bf16", 30.0, "index", "none", 0, True, False),
        # patches packed into sequences, each attending to itself, grid distance in the scores, training step
        _attention("attention packed train", 2, 4096, 4096, 8, 8, 64, "bf16", 0.0, "grid", "none", 16, False, True),
        # long series: a known prefix seen by all, the rest in order; capped scores, shared heads; training step
        _attention("attention prefix train", 1, 8192, 8192, 8, 2, 128, "bf16", 50.0, "none", "prefix", 0, False, True),
        # the float32 network on single 16x16 maps, training step
        _attention("attention maps f32 train", 16, 256, 256, 4, 4, 32, "f32", 0.0, "grid", "none", 0, False, True),
        # an odd length and width in float16, in order
        _attention("attention odd f16", 3, 1999, 1999, 6, 3, 80, "f16", 20.0, "index", "causal", 0, True, False),
    ]


def _span(rng, lo, hi):
    """A whole number of [lo, hi], even over the logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw(rng):
    kind = rng.choice(("norm", "norm", "rotary", "attention", "attention", "attention"))
    dtype = rng.choice(("f32", "bf16", "bf16", "f16"))
    if kind == "norm":
        out, train = rng.choice((dtype, "bf16", "f32")), rng.random() < 0.6
        if rng.random() < 0.5:
            return _norm(None, "rows", _span(rng, 1, 65536), _span(rng, 32, 9000), 1, dtype, out, train, train)
        n, points = rng.choice(((243, 256), (1251, 16), (243, 1024), (8932, 16), (_span(rng, 50, 9000), _span(rng, 4, 1024))))
        return _norm(None, "maps", _span(rng, 1, 1024), n, points, "f32", out, train, train and rng.random() < 0.5)
    if kind == "rotary":
        dim = 2 * _span(rng, 8, 64)
        pairs = dim // 2 - rng.choice((0, 0, rng.randrange(dim // 4)))
        time = rng.randrange(pairs // 2)
        rows = rng.randrange(1, pairs - time)
        kv = rng.choice((1, 2, 4))
        return _rotary(None, _span(rng, 1, 64), _span(rng, 1, 8192), kv * rng.choice((1, 2, 3, 4)), kv, dim, time, rows,
                       pairs - time - rows, rng.random() < 0.5, dtype, rng.random() < 0.5)
    dim, kv = rng.choice((16, 32, 40, 64, 64, 80, 96, 128, 128)), rng.choice((1, 2, 4))
    heads = kv * rng.choice((1, 1, 2, 3, 4))
    cap, bias = rng.choice((0.0, 0.0, 20.0, 50.0)), rng.choice(("none", "index", "grid"))
    if rng.random() < 0.4:
        return _attention(None, _span(rng, 1, 128), rng.choice((1, 1, 1, 2, 5)), _span(rng, 16, 32768), heads, kv, dim, dtype, cap,
                          bias, rng.choice(("none", "causal")), rng.choice((0, 0, 3)), rng.random() < 0.7, False)
    t = _span(rng, 17, 8192)
    return _attention(None, _span(rng, 1, 32), t, t, heads, kv, dim, dtype, cap, bias, rng.choice(("none", "causal", "prefix")),
                      rng.choice((0, 0, max(1, t // 256))), rng.random() < 0.3, rng.random() < 0.6)


def _cost(case):
    """Rough cost of the plain form: bytes and the score matrices that it makes."""
    w = work(case)
    scores = case["batch"] * case["heads"] * case["tq"] * case["tk"] if case["op"] == "attention" else 0
    return w["bytes"] + w["flops"] / 64 + scores * (80 if case["train"] else 40)


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "rotary", "attention")}
    while True:
        case = _draw(rng)
        if _cost(case) <= most[case["op"]]:
            return case


# ----------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _grid_positions(index):
    """(time, row, column) of the index-th position of a series of GRID x GRID maps, int32."""
    return torch.stack((index // (GRID * GRID), index // GRID % GRID, index % GRID), -1).to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["op"] == "norm":
        n, lead, points = case["n"], case["lead"], case["points"]
        # coefficients are non-negative and their scales spread over three orders of magnitude
        scale = torch.exp(_randn(g, n) * 1.5 - 3)
        if case["layout"] == "maps":
            maps = (_randn(g, lead, n, points).mul_(0.4).add_(1).abs_()).mul_(scale[:, None])
            x = maps.transpose(1, 2)                       # (lead, points, n): tokens, read where the maps lie
        else:
            x = (_randn(g, lead, n).mul_(0.4).add_(1)).mul_(scale).to(DTYPES[case["dtype"]])
        s["x"] = x.detach().requires_grad_(case["x_grad"])
        s["weight"] = (1 + 0.2 * _randn(g, n)).requires_grad_(case["train"])
        s["bias"] = (0.1 * _randn(g, n)).requires_grad_(case["train"])
        if case["train"]:
            s["dy"] = _randn(g, *x.shape).to(DTYPES[case["out"]])
        return s
    dtype = DTYPES[case["dtype"]]
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        t = case["tokens"]
        # the projection's output, q beside k in one row of it
        qk = _randn(g, b, t, h + kv, d).to(dtype)
        s["q"] = qk[:, :, :h].detach().requires_grad_(case["train"])
        s["k"] = qk[:, :, h:].detach().requires_grad_(case["train"])
        start = torch.randint(0, 200000, (b, 1), generator=g, device="cuda")
        s["positions"] = _grid_positions(start + torch.arange(t, device="cuda"))
        if case["train"]:
            s["dq"], s["dk"] = _randn(g, b, t, h, d).to(dtype), _randn(g, b, t, kv, d).to(dtype)
        return s
    tq, tk = case["tq"], case["tk"]
    q = _randn(g, b, tq, h, d) * (2.0 if case["cap"] else 1.0)
    s["q"] = q.to(dtype).requires_grad_(case["train"])
    s["k"] = _randn(g, b, tk, kv, d).to(dtype).requires_grad_(case["train"])
    s["v"] = _randn(g, b, tk, kv, d).to(dtype).requires_grad_(case["train"])
    lengths = None
    if case["ragged"]:
        lengths = torch.randint((tk + 1) // 2, tk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    s["k_lengths"] = lengths
    index = torch.arange(tk, device="cuda").expand(b, tk)
    document = None
    # where the queries stand among the keys: the whole sequence, or the newest of what is stored
    newest = torch.arange(tk, device="cuda").expand(b, tk)
    if tq < tk:
        last = torch.full((b,), tk, device="cuda") if lengths is None else lengths.long()
        newest = (last[:, None] - tq + torch.arange(tq, device="cuda")).clamp(min=0)
    if case["documents"]:
        # borders anywhere; in packed sequences the last twentieth is left empty
        edge = torch.rand(b, case["documents"] - 1, generator=g, device="cuda").mul_(0.95 * tk).long().sort(1)[0]
        document = torch.searchsorted(edge, index.contiguous(), right=True)
        first = torch.cat((torch.zeros_like(edge[:, :1]) if edge.shape[1] else edge.new_zeros(b, 1), edge), 1)
        index = index - first.gather(1, document)
        empty = torch.arange(tk, device="cuda") >= (max(1, int(0.95 * tk)) if tq == tk else tk)
        document = document.masked_fill(empty, -1).to(torch.int32)
    s["k_documents"] = document
    s["q_documents"] = None if document is None else document.gather(1, newest)
    s["k_positions"] = s["q_positions"] = s["slopes"] = s["prefix"] = None
    if case["bias"] != "none":
        s["slopes"] = (2.0 ** -(1 + 7 * torch.rand(h, generator=g, device="cuda"))).requires_grad_(case["train"])
    if case["bias"] == "grid":
        s["k_positions"] = _grid_positions(index)
        s["q_positions"] = _grid_positions(index.gather(1, newest))
    if case["mask"] == "prefix":
        s["prefix"] = torch.randint(tk // 8, tk // 4 + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    if case["train"]:
        s["do"] = _randn(g, b, tq, h, d).to(dtype)
    return s


# ------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, weight, bias, out):
    x = x.float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    scaled = centred * torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    return (scaled * weight + bias).to(out)


def _angles(positions, sections):
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=positions.device)
    power = torch.tensor([i / n for n in sections for i in range(n)], device=positions.device, dtype=torch.float64)
    return positions.double()[..., axis] * BASE ** -power


def _plain_rotary(x, angles, interleaved):
    n = angles.shape[-1]
    cos, sin = angles.cos().float().unsqueeze(-2), angles.sin().float().unsqueeze(-2)
    y = x.float()
    turn, rest = y[..., : 2 * n], y[..., 2 * n:]
    if interleaved:
        x0, x1 = turn[..., 0::2], turn[..., 1::2]
        turned = torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2)
    else:
        x0, x1 = turn[..., :n], turn[..., n:]
        turned = torch.cat((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1)
    return torch.cat((turned, rest), -1).to(x.dtype)


def _visible(s):
    """(batch, 1, tq, tk) truth values, or None where every query sees every key."""
    case = s["case"]
    tq, tk = case["tq"], case["tk"]
    dev = s["q"].device
    key = torch.arange(tk, device=dev)
    length = torch.full((case["batch"],), tk, device=dev) if s["k_lengths"] is None else s["k_lengths"].long()
    see = None
    if s["k_lengths"] is not None:
        see = (key < length[:, None])[:, None, None, :]
    if case["mask"] != "none":
        query = torch.arange(tq, device=dev) + (length[:, None] - tq)
        order = key <= query[..., None]
        if s["prefix"] is not None:
            order = order | (key < s["prefix"][:, None, None])
        see = order[:, None] if see is None else see & order[:, None]
    if s["k_documents"] is not None:
        qd, kd = s["q_documents"], s["k_documents"]
        same = (qd[:, :, None] == kd[:, None, :]) & (qd[:, :, None] >= 0)
        see = same[:, None] if see is None else see & same[:, None]
    return see


def _distance(s):
    """(batch, 1, tq, tk) whole numbers in float32."""
    case = s["case"]
    if s["k_positions"] is not None:
        return (s["q_positions"][:, :, None] - s["k_positions"][:, None]).abs().sum(-1)[:, None].float()
    dev = s["q"].device
    length = torch.full((case["batch"],), case["tk"], device=dev) if s["k_lengths"] is None else s["k_lengths"].long()
    query = torch.arange(case["tq"], device=dev) + (length[:, None] - case["tq"])
    return (query[..., None] - torch.arange(case["tk"], device=dev)).abs()[:, None].float()


def _plain_attention(s):
    case, q = s["case"], s["q"]
    group = case["heads"] // case["kv_heads"]
    qh = q.float().transpose(1, 2)
    kh = s["k"].float().transpose(1, 2).repeat_interleave(group, 1)
    vh = s["v"].float().transpose(1, 2).repeat_interleave(group, 1)
    z = torch.matmul(qh, kh.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(case["dim"]))
    if case["cap"]:
        z = case["cap"] * torch.tanh(z / case["cap"])
    if s["slopes"] is not None:
        z = z - s["slopes"][:, None, None] * _distance(s)
    see = _visible(s)
    if see is not None:
        z = z.masked_fill(~see, -math.inf)
    top = z.detach().amax(-1, keepdim=True)
    p = torch.exp(z - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(-1, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    return torch.matmul(p, vh).transpose(1, 2).to(q.dtype)


def run(state):
    s, case = state, state["case"]
    if own:
        from wst_amd import tokens
    if case["op"] == "norm":
        out = DTYPES[case["out"]]
        if own:
            y = tokens.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, out_dtype=out)
        else:
            y = _plain_norm(s["x"], s["weight"], s["bias"], out)
        if not case["train"]:
            return y
        leaves = ([s["x"]] if case["x_grad"] else []) + [s["weight"], s["bias"]]
        return (y.detach(), *torch.autograd.grad(y, leaves, s["dy"]))
    if case["op"] == "rotary":
        sections = (case["time"], case["rows"], case["cols"])
        if own:
            q, k = tokens.rotary(s["q"], s["positions"], sections, base=BASE, interleaved=case["interleaved"], k=s["k"])
        else:
            angles = _angles(s["positions"], sections)
            q, k = _plain_rotary(s["q"], angles, case["interleaved"]), _plain_rotary(s["k"], angles, case["interleaved"])
        if not case["train"]:
            return q, k
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if own:
        o = tokens.attention(s["q"], s["k"], s["v"], cap=case["cap"], slopes=s["slopes"], q_positions=s["q_positions"],
                             k_positions=s["k_positions"], q_documents=s["q_documents"], k_documents=s["k_documents"],
                             causal=case["mask"] == "causal", prefix=s["prefix"], k_lengths=s["k_lengths"])
    else:
        o = _plain_attention(s)
    if not case["train"]:
        return o.detach()
    leaves = [s["q"], s["k"], s["v"]] + ([] if s["slopes"] is None else [s["slopes"]])
    return (o.detach(), *torch.autograd.grad(o, leaves, s["do"]))


# ------------------------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "norm":
        n, values = case["n"], case["lead"] * case["points"] * case["n"]
        moved, flops = values * (size[case["dtype"]] + size[case["out"]]) + 8 * n, 8 * values
        if case["train"]:
            # the step reads x and dy (x counts once) and writes the gradients
            moved += values * (size[case["out"]] + (size[case["dtype"]] if case["x_grad"] else 0)) + 8 * n
            flops += (14 if case["x_grad"] else 5) * values
        return {"bytes": moved, "flops": flops}
    b, h, kv, d, e = case["batch"], case["heads"], case["kv_heads"], case["dim"], size[case["dtype"]]
    if case["op"] == "rotary":
        values = b * case["tokens"] * (h + kv) * d
        times = 2 if case["train"] else 1
        return {"bytes": 2 * times * values * e + 12 * b * case["tokens"], "flops": 3 * times * values}
    tq, tk = case["tq"], case["tk"]
    keys = tk * (0.75 if case["ragged"] else 1.0)
    pairs = tq * keys
    if case["mask"] == "causal":
        pairs = tq * (keys - (tq - 1) / 2)
    if case["mask"] == "prefix":
        pairs = tq * keys / 2 + (keys * 3 / 16) ** 2 / 2
    if case["documents"]:
        pairs *= 0.9 / max(1, case["documents"]) if tq == tk else 1.0 / case["documents"]
    moved = e * d * b * (2 * h * tq + 2 * kv * keys)
    flops = 4 * d * pairs * b * h
    if case["train"]:
        moved += e * d * b * (2 * h * tq + 2 * kv * keys)
        flops += 10 * d * pairs * b * h
    return {"bytes": int(moved), "flops": int(max(flops, 1))}


# ------------------------------------------------------------------------------------------------ exact
def _exact_norm(s):
    case = s["case"]
    x = s["x"].detach().double().reshape(-1, case["n"])
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    dev, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    r = 1.0 / torch.sqrt(dev + EPS)
    h = x.sub_(mean).mul_(r)
    shape = s["x"].shape
    y = torch.addcmul(b, h, w).reshape(shape)
    if not case["train"]:
        return y
    dy = s["dy"].double().reshape(-1, case["n"])
    dw, db = (dy * h).sum(0), dy.sum(0)
    if not case["x_grad"]:
        return y, dw, db
    g = dy.mul_(w)
    m0, m1 = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    return y, g.sub_(m0).sub_(h.mul_(m1)).mul_(r).reshape(shape), dw, db


def _exact_rotary(s):
    case = s["case"]
    sections = (case["time"], case["rows"], case["cols"])
    n = sum(sections)

    def turned(x, sign):
        y = x.detach().double().clone()
        p = 0
        for axis, count in enumerate(sections):
            for i in range(count):
                angle = s["positions"][..., axis].double() * (BASE ** (-i / count)) * sign
                turn = torch.polar(torch.ones_like(angle), angle)[..., None]
                at, to = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + n)
                z = torch.complex(y[..., at], y[..., to]) * turn
                y[..., at], y[..., to] = z.real, z.imag
                p += 1
        return y

    both = (turned(s["q"], 1.0), turned(s["k"], 1.0))
    return both if not case["train"] else both + (turned(s["dq"], -1.0), turned(s["dk"], -1.0))


def _exact_attention(s):
    """One sequence and head at a time, the gradients from their formulas."""
    case = s["case"]
    if case["batch"] * case["heads"] * case["tq"] * case["tk"] > 3e9:
        return None
    q, k, v = (s[x].detach().double() for x in "qkv")
    o, scale, group = torch.zeros_like(q), case["dim"] ** -0.5, case["heads"] // case["kv_heads"]
    train = case["train"]
    if train:
        do, dq, dk, dv = s["do"].double(), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dslopes = torch.zeros(case["heads"], dtype=torch.float64, device=q.device)
    i, j = torch.arange(case["tq"], device=q.device)[:, None], torch.arange(case["tk"], device=q.device)[None]
    for b in range(case["batch"]):
        end = case["tk"] if s["k_lengths"] is None else int(s["k_lengths"][b])
        at = i + end - case["tq"]
        hidden = (j >= end).expand(case["tq"], case["tk"])
        if case["mask"] != "none":
            late = j > at
            if s["prefix"] is not None:
                late = late & (j >= int(s["prefix"][b]))
            hidden = hidden | late
        if s["k_documents"] is not None:
            qd, kd = s["q_documents"][b], s["k_documents"][b]
            hidden = hidden | (qd[:, None] != kd[None]) | (kd[None] < 0)
        far = None
        if s["k_positions"] is not None:
            far = sum((s["q_positions"][b, :, a].double()[:, None] - s["k_positions"][b, :, a].double()[None]).abs() for a in range(3))
        elif s["slopes"] is not None:
            far = (at - j).abs().double()
        for h in range(case["heads"]):
            c = h // group
            z = q[b, :, h] @ k[b, :, c].T * scale
            t = torch.tanh(z / case["cap"]) if case["cap"] else None
            z = z if t is None else case["cap"] * t
            if far is not None:
                z = z - s["slopes"][h].double() * far
            z = torch.where(hidden, torch.full_like(z, -math.inf), z)
            p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
            o[b, :, h] = p @ v[b, :, c]
            if train:
                dp = do[b, :, h] @ v[b, :, c].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                if far is not None:
                    dslopes[h] -= (ds * far).sum()
                if t is not None:
                    ds = ds * (1 - t * t)
                dq[b, :, h] = ds @ k[b, :, c] * scale
                dk[b, :, c] += ds.T @ q[b, :, h] * scale
                dv[b, :, c] += p.T @ do[b, :, h]
    if not train:
        return o
    return (o, dq, dk, dv) + (() if s["slopes"] is None else (dslopes,))


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "rotary": _exact_rotary, "attention": _exact_attention}[case["op"]](s)

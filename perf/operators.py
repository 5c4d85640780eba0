"""What the operators around a neighborhood-attention layer are measured on: the
norm in front of it (and on its queries and keys), rotary positions by axis, and
the serving step against cached keys whose prefix the whole batch shares.

A case is a dict of plain values; ``op`` names the entry point:

* ``norm``   -- ``layer_norm``; ``step``: with the gradients of input, weight and
  bias.  ``packed`` > 0: the rows are one of the ``packed`` parts of a
  projection's output ``[rows / heads, packed, heads, channels]``;
* ``rotary`` -- ``rotary`` of queries and keys; ``step``: with their gradients.
  ``spatial`` is a text such as ``"16x32x32"``.  ``positions``: ``"grid"`` (the
  tokens' own coordinates) or the type of a tensor of ``axes`` coordinates per
  token.  ``dims``: rotated channels per axis, such as ``"16x24x24"``;
* ``prefix`` -- ``prefix_attention``: ``tokens`` new tokens of every sample
  against ``prefix`` shared tokens and a cache of up to ``cache`` own ones
  (``window`` > 0: the last ``window`` of them only).

Plain forms are elementary torch operations in float32 (angles in float64).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
POSITIONS = {"i64": torch.int64, "i32": torch.int32, "f32": torch.float32}
EPS = 1e-5
THETA = 10000.0


def _norm(name, dtype, rows, channels, heads=1, packed=0, step=True, wide=False):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "channels": channels,
            "heads": heads, "packed": packed, "step": step, "wide_weights": wide}


def _rotary(name, dtype, batch, spatial, heads, kv_heads, dim, dims, positions="grid",
            interleaved=False, step=True):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "spatial": spatial,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dims": dims,
            "positions": positions, "interleaved": interleaved, "step": step}


def _prefix(name, dtype, batch, heads, kv_heads, dim, prefix, cache, tokens=1, window=0):
    return {"name": name, "op": "prefix", "dtype": dtype, "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "prefix": prefix, "cache": cache,
            "tokens": tokens, "window": window}


def listed():
    return [
        # the norm of one generated token: the call itself is the cost
        _norm("norm token bf16", "bf16", 1, 256, step=False),
        # the norm before a layer of an image model's stage, in training
        _norm("norm image step bf16", "bf16", 8 * 56 * 56, 256),
        # the queries of a packed projection normalised per head, single-precision weights
        _norm("norm heads step f16", "f16", 4 * 56 * 56 * 4, 32, heads=4, packed=3, wide=True),
        # torch's default type, a width that no vector divides
        _norm("norm odd step f32", "f32", 5115, 1001),
        # long sequences of a wide model
        _norm("norm wide step bf16", "bf16", 65536, 2048),
        # video tokens, rotated by time, height and width, in training
        _rotary("rotary video step bf16", "bf16", 2, "16x64x64", 8, 8, 64, "16x24x24"),
        # one new token of each request, far positions on three axes
        _rotary("rotary token bf16", "bf16", 64, "1", 32, 8, 128, "32x48x48", positions="i64",
                step=False),
        # a text sequence in single precision: adjacent pairs, part of the channels, odd length
        _rotary("rotary sequence step f32", "f32", 3, "4097", 6, 3, 40, "24", interleaved=True),
        # a small service: few requests, short prefix, odd lengths
        _prefix("prefix token small bf16", "bf16", 4, 8, 2, 64, 1001, 251),
        # a chat service: a long system prompt, each request's own turns
        _prefix("prefix token bf16", "bf16", 32, 32, 8, 128, 16384, 2048),
        # the same under load, a long shared document
        _prefix("prefix token large f16", "f16", 64, 32, 8, 128, 65536, 2048),
        # chunks of prompts behind a shared prefix, sliding windows over the own tokens
        _prefix("prefix chunk bf16", "bf16", 8, 16, 4, 64, 8192, 640, tokens=128, window=255),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_norm(rng):
    heads, packed = 1, 0
    if rng.random() < 0.3:  # a head of a packed projection
        heads, packed, channels = rng.randint(1, 16), 3, 8 * rng.randint(1, 16)
    elif rng.random() < 0.5:
        channels = 8 * _log(rng, 1, 2048)
    else:
        channels = _log(rng, 5, 16384)
    rows = _log(rng, 1, min(262144, (1 << 27) // channels))
    rows = -(-rows // heads) * heads
    return _norm("", rng.choice(list(DTYPES)), rows, channels, heads, packed,
                 rng.random() < 0.7, rng.random() < 0.3)


def _draw_rotary(rng):
    axes = rng.randint(1, 3)
    pairs = rng.choice((16, 20, 32, 36, 48, 64))
    cuts = sorted(rng.randint(1, pairs) for _ in range(axes))
    dims = [2 * max(1, b - a) for a, b in zip([0] + cuts, cuts)]
    dim = 2 * max(pairs, sum(dims) // 2)
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 1, 2, 4))
    total = _log(rng, 1, max(1, (1 << 25) // (dim * (heads + kv_heads))))
    batch = min(total, _log(rng, 1, 64))
    positions = rng.choice(("grid", "grid", "i64", "i32", "f32"))
    left, spatial = max(1, total // batch), []
    for a in range(axes - 1 if positions == "grid" else 0):
        spatial.append(max(1, _log(rng, 1, max(1, left)) // 2))
        left = max(1, left // spatial[-1])
    spatial.append(left)
    return _rotary("", rng.choice(list(DTYPES)), batch, "x".join(map(str, spatial)), heads,
                   kv_heads, dim, "x".join(map(str, dims)), positions, rng.random() < 0.4,
                   rng.random() < 0.6)


def _draw_prefix(rng):
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    dim = rng.choice((32, 40, 64, 64, 80, 96, 128, 128, 256))
    tokens = 1 if rng.random() < 0.6 else _log(rng, 2, 130)
    batch = _log(rng, 1, 64)
    while batch * tokens * heads > 8192:
        batch, tokens = -(-batch // 2), -(-tokens // 2)
    most = (1 << 27) // (batch * tokens * heads)  # scores of a pass
    prefix = _log(rng, 1, min(65536, most)) if rng.random() < 0.9 else 0
    cache = _log(rng, 1, min(2048, most))
    window = _log(rng, 1, cache) if rng.random() < 0.3 else 0
    return _prefix("", rng.choice(("bf16", "f16", "bf16", "f16", "f32")), batch, heads, kv_heads,
                   dim, prefix, cache, tokens, window)


def draw(rng):
    case = rng.choice((_draw_norm, _draw_rotary, _draw_prefix))(rng)
    del case["name"]
    return case


def _ints(text):
    return tuple(int(x) for x in text.split("x"))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0, mean=0.0, dt=dtype):
        return torch.randn(shape, generator=g, device=DEVICE).mul_(std).add_(mean).to(dt)

    s = {"op": case["op"]}
    if case["op"] == "norm":
        rows, c, h = case["rows"], case["channels"], case["heads"]
        if case["packed"]:
            x = randn(rows // h, case["packed"], h, c, std=1.5, mean=0.3)[:, 0]
        else:
            x = randn(rows, c, std=1.5, mean=0.3)
        wt = torch.float32 if case["wide_weights"] else dtype
        s.update(x=x, w=randn(c, std=0.2, mean=1.0, dt=wt), b=randn(c, std=0.2, dt=wt),
                 step=case["step"])
        leaves = ("x", "w", "b")
        if case["step"]:
            s["g"] = randn(*x.shape)
    elif case["op"] == "rotary":
        spatial, dims = _ints(case["spatial"]), _ints(case["dims"])
        lead = (case["batch"], *spatial)
        s.update(q=randn(*lead, case["heads"], case["dim"]),
                 k=randn(*lead, case["kv_heads"], case["dim"]), dims=dims, step=case["step"],
                 interleaved=case["interleaved"], positions=None)
        if case["positions"] != "grid":
            # image and video tokens inside texts: up to a million positions on
            s["positions"] = torch.randint(0, 1 << 20, (*lead, len(dims)), generator=g,
                                           device=DEVICE).to(POSITIONS[case["positions"]])
        leaves = ("q", "k")
        if case["step"]:
            s["gq"], s["gk"] = randn(*s["q"].shape), randn(*s["k"].shape)
    else:
        b, hk, d = case["batch"], case["kv_heads"], case["dim"]
        s.update(q=randn(b, case["tokens"], case["heads"], d, std=1.5),
                 pk=randn(case["prefix"], hk, d), pv=randn(case["prefix"], hk, d),
                 k=randn(b, case["cache"], hk, d), v=randn(b, case["cache"], hk, d),
                 lens=torch.randint(0, case["cache"] + 1, (b,), generator=g, device=DEVICE,
                                    dtype=torch.int32),
                 window=case["window"] or None)
        leaves = ()
    if case.get("step"):
        for n in leaves:
            s[n].requires_grad_(True)
    return s


# ---- the framework's calls ---------------------------------------------------

def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "natten-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import natten_amd

    return natten_amd


def _run_own(s):
    natten_amd = sys.modules.get("natten_amd") or _package()
    if s["op"] == "norm":
        y = natten_amd.layer_norm(s["x"], s["w"], s["b"], EPS)
        if not s["step"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["g"]))
    if s["op"] == "rotary":
        q, k = natten_amd.rotary(s["q"], s["k"], positions=s["positions"], axis_dims=s["dims"],
                                 theta=THETA, interleaved=s["interleaved"])
        if not s["step"]:
            return q, k
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["gq"], s["gk"]))
        return q.detach(), k.detach(), dq, dk
    return natten_amd.prefix_attention(s["q"], s["pk"], s["pv"], s["k"], s["v"],
                                       seq_lens=s["lens"], kernel_size=s["window"],
                                       return_lse=True)


# ---- plain forms -------------------------------------------------------------

def _plain_norm(s):
    x, w, b = s["x"].float(), s["w"].float(), s["b"].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if not s["step"]:
        return y
    g = s["g"].float()
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return (y, dx.to(s["x"].dtype), (g * xh).sum(rows).to(s["w"].dtype),
            g.sum(rows).to(s["b"].dtype))


def _grid(lead):
    axes = [torch.arange(n, device=DEVICE, dtype=torch.float64) for n in lead[1:]]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1)


def _plain_rotary(s):
    q, dims = s["q"], s["dims"]
    pos = _grid(q.shape[:-2]) if s["positions"] is None else s["positions"].double()
    dev, total = q.device, sum(dims)
    # per rotated pair: its axis, its frequency, its two channels
    axis = torch.cat([torch.full((d // 2,), a, device=dev) for a, d in enumerate(dims)])
    freq = torch.cat([THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
                      for d in dims])
    first = [sum(dims[:a]) for a in range(len(dims))]
    step = 2 if s["interleaved"] else 1
    u = torch.cat([f + step * torch.arange(d // 2, device=dev) for f, d in zip(first, dims)])
    v = u + 1 if s["interleaved"] else u + torch.tensor(
        [d // 2 for d in dims], device=dev)[axis]
    angle = (pos[..., axis] * freq).unsqueeze(-2)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x, sn):
        xf = x.float()
        xu, xv = xf[..., u], xf[..., v]
        out = xf.clone()
        out[..., u] = xu * cos - xv * sn
        out[..., v] = xu * sn + xv * cos
        return out.to(x.dtype)

    assert total <= q.shape[-1]
    with torch.no_grad():
        out = (turn(q, sin), turn(s["k"], sin))
        if not s["step"]:
            return out
        return (*out, turn(s["gq"], -sin), turn(s["gk"], -sin))


def _plain_prefix(s):
    q, hk = s["q"], s["pk"].shape[1]
    b, lq, h, d = q.shape
    n, cap, rep = s["pk"].shape[0], s["k"].shape[1], h // hk
    scale = d ** -0.5
    qf = q.float().view(b, lq, hk, rep, d).permute(2, 0, 1, 3, 4).contiguous()
    pk, pv = (t.float().permute(1, 2, 0).contiguous() for t in (s["pk"], s["pv"]))
    k, v = (t.float().permute(2, 0, 3, 1).contiguous() for t in (s["k"], s["v"]))
    s1 = torch.matmul(qf.view(hk, b * lq * rep, d), pk).view(hk, b, lq * rep, n) * scale
    s2 = torch.matmul(qf.view(hk, b, lq * rep, d), k).view(hk, b, lq, rep, cap) * scale
    tok = s["lens"].view(b, 1, 1, 1).long() - lq + torch.arange(
        lq, device=q.device).view(1, lq, 1, 1)
    pos = torch.arange(cap, device=q.device)
    seen = pos <= tok
    if s["window"]:
        seen &= pos > tok - s["window"]
    s2 = s2.masked_fill(~seen, -math.inf).view(hk, b, lq * rep, cap)
    scores = torch.cat((s1, s2), -1)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p[..., :n].reshape(hk, b * lq * rep, n),
                     pv.transpose(1, 2).contiguous()).view(hk, b, lq * rep, d)
    o = o + torch.matmul(p[..., n:].contiguous(), v.transpose(2, 3).contiguous())
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = top + torch.log(total)
    o = o.view(hk, b, lq, rep, d).permute(1, 2, 0, 3, 4).reshape(b, lq, h, d)
    lse = lse.view(hk, b, lq, rep).permute(1, 2, 0, 3).reshape(b, lq, h)
    return o.to(q.dtype), lse


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "rotary": _plain_rotary,
                "prefix": _plain_prefix}[state["op"]](state)


# ---- work --------------------------------------------------------------------

def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, c = case["rows"] * case["channels"], case["channels"]
        wb = 4 if case["wide_weights"] else e
        if case["step"]:
            return {"bytes": 4 * n * e + 4 * c * wb, "flops": 22 * n}
        return {"bytes": 2 * n * e + 2 * c * wb, "flops": 8 * n}
    if case["op"] == "rotary":
        tokens = case["batch"] * math.prod(_ints(case["spatial"]))
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        pos = {"grid": 0, "i64": 8, "i32": 4, "f32": 4}[case["positions"]]
        passes = 2 if case["step"] else 1
        return {"bytes": 2 * passes * n * e + tokens * len(_ints(case["dims"])) * pos,
                "flops": 3 * passes * n}
    rows = case["batch"] * case["tokens"] * case["heads"]
    # lengths are drawn evenly between none and the whole cache
    held = seen = case["cache"] / 2
    if case["window"]:
        held = min(held, case["window"] + case["tokens"] - 1)
        seen = min(seen, case["window"])
    kv = (case["prefix"] + case["batch"] * held) * case["kv_heads"] * case["dim"]
    return {"bytes": 2 * rows * case["dim"] * e + rows * 4 + 2 * kv * e,
            "flops": 4 * rows * case["dim"] * (case["prefix"] + seen)}


# ---- values in 64 bits, from the definitions ---------------------------------

def _exact_norm(s):
    x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    flat = x.reshape(-1, x.shape[-1])
    var, mean = torch.var_mean(flat, 1, correction=0, keepdim=True)
    unit = (flat - mean) * torch.rsqrt(var + EPS)
    y = torch.addcmul(b, unit, w).view(x.shape)
    if not s["step"]:
        return y
    g = s["g"].double().reshape(flat.shape)
    # the gradient is what is left of g w / std without its parts along 1 and unit
    t = g * w
    along = (t * unit).sum(1, keepdim=True) / flat.shape[1]
    dx = (t - t.mean(1, keepdim=True) - along * unit) * torch.rsqrt(var + EPS)
    return y, dx.view(x.shape), (unit * g).sum(0), g.sum(0)


def _exact_rotary(s):
    q, dims, lead = s["q"], s["dims"], s["q"].shape[:-2]
    parts, first = [], 0
    pos = _grid(lead).expand(*lead, -1) if s["positions"] is None else s["positions"].double()
    for a, d in enumerate(dims):
        rate = torch.exp(torch.arange(d // 2, device=q.device, dtype=torch.float64)
                         * (-2.0 * math.log(THETA) / d))
        parts.append((first, d, torch.polar(torch.ones((), dtype=torch.float64, device=q.device),
                                            pos[..., a, None] * rate).unsqueeze(-2)))
        first += d

    def turn(x, back):
        out = x.detach().double().clone()
        for f, d, z in parts:
            part = out[..., f:f + d].clone()
            if s["interleaved"]:
                c = torch.complex(part[..., 0::2], part[..., 1::2])
            else:
                c = torch.complex(part[..., :d // 2].contiguous(), part[..., d // 2:].contiguous())
            c = c * (z.conj() if back else z)
            if s["interleaved"]:
                out[..., f:f + d:2], out[..., f + 1:f + d:2] = c.real, c.imag
            else:
                out[..., f:f + d] = torch.cat((c.real, c.imag), -1)
        return out

    out = (turn(q, False), turn(s["k"], False))
    if not s["step"]:
        return out
    return (*out, turn(s["gq"], True), turn(s["gk"], True))


def _exact_prefix(s):
    q = s["q"].double()
    b, lq, h, d = q.shape
    hk = s["pk"].shape[1]
    rep = h // hk
    out, lse = torch.zeros_like(q), torch.full(q.shape[:-1], -math.inf, dtype=torch.float64,
                                               device=q.device)
    lens = s["lens"].tolist()
    pk, pv = (s[n].double().transpose(0, 1).contiguous() for n in ("pk", "pv"))
    n = pk.shape[1]
    for i in range(b):  # one request at a time, its tokens cut to their number
        m = lens[i]
        keys = torch.cat((pk, s["k"][i, :m].double().transpose(0, 1)), 1)
        vals = torch.cat((pv, s["v"][i, :m].double().transpose(0, 1)), 1)
        if keys.shape[1] == 0:
            continue
        x = q[i].view(lq, hk, rep, d).permute(1, 0, 2, 3).reshape(hk, lq * rep, d)
        z = torch.matmul(x, keys.transpose(1, 2).contiguous()).view(hk, lq, rep, -1) / math.sqrt(d)
        at = torch.arange(n + m, device=q.device) - n
        t = (m - lq + torch.arange(lq, device=q.device)).view(lq, 1, 1)
        hide = at > t
        if s["window"]:
            hide = hide | (at <= t - s["window"])
        hide = hide & (at >= 0)
        z = z.masked_fill(hide, -math.inf)
        l = torch.logsumexp(z, -1)
        p = torch.exp(z - torch.where(l == -math.inf, torch.zeros_like(l), l).unsqueeze(-1))
        o = torch.matmul(p.view(hk, lq * rep, -1), vals).view(hk, lq, rep, d)
        out[i] = o.permute(1, 0, 2, 3).reshape(lq, h, d)
        lse[i] = l.permute(1, 0, 2).reshape(lq, h)
    return out, lse


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "rotary": _exact_rotary,
                "prefix": _exact_prefix}[case["op"]](s)

"""norm_rotary against its formula in float64, forward and backward: every way that
lanes share a row, grids and tensors of positions, views, missing keys, weights and
gradients, both implementations of the node, special rows, streams and graph
capture; layers that use it; and what it refuses.

Tolerances.  With e = 2^-24 (half a step of float32) and rows of at most 256 channels,
K = 64 bounds the relative error of a sum against the sum of magnitudes and of the
few operations after it (16 sequential and 6 pairwise additions).  |xh| is off by at
most ex = K e (|xh| + rstd max|x|), the normed row z by tz = |w| ex + K e (|w xh| + |b|).
A rotation adds 8 e (|u| + |v|) to what its two channels are off by (test_rotary).  So y
is off by tz_u + tz_v + 8 e (|z_u| + |z_v|), g' = R^T g by tg = 8 e (|g_u| + |g_v|); dx by
rstd times (K e of its terms' magnitudes, what ex moves them by, and tg through the
same sums); dw adds `rows` terms: (rows + K) e sum|g' xh| + sum(|g'| ex + tg |xh|).  Each
plus half a step of the result's own type.
"""

import math

import pytest
import torch

from _helpers import DEV, randn
from test_rotary import _grid

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E, K = 2.0 ** -24, 64
NAMES = ("q", "k", "wq", "bq", "wk", "bk")


def _half(t, dtype):
    return t.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny


def _pairs(dims, interleaved):
    """Channels of each rotated pair, its axis and its rate's exponent."""
    u, v, axis, power, first = [], [], [], [], 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            u.append(first + (2 * i if interleaved else i))
            v.append(first + (2 * i + 1 if interleaved else i + d // 2))
            axis.append(a)
            power.append(-2.0 * i / d)
        first += d
    return u, v, axis, power


def _turn(x, t, pos, dims, theta, interleaved, sign):
    """x off by t, turned: the value and how far off it may be."""
    u, v, axis, power = _pairs(dims, interleaved)
    angle = (sign * pos[..., axis] * theta ** torch.tensor(power, dtype=torch.float64)).unsqueeze(-2)
    out, tol = x.clone(), t.clone()
    xu, xv = x[..., u], x[..., v]
    out[..., u] = xu * angle.cos() - xv * angle.sin()
    out[..., v] = xu * angle.sin() + xv * angle.cos()
    tol[..., u] = tol[..., v] = t[..., u] + t[..., v] + 8 * E * (xu.abs() + xv.abs())
    return out, tol


def _formula(x, w, b, g, pos, dims, theta, interleaved, eps):
    """{y, dx, dw, db} of one of the tensors, each (value, tolerance)."""
    xd = x.double()
    d = x.shape[-1]
    wd = torch.ones(d, dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(d, dtype=torch.float64) if b is None else b.double()
    xc = xd - xd.mean(-1, keepdim=True)
    rstd = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xc * rstd
    ex = K * E * (xh.abs() + rstd * xd.abs().amax(-1, keepdim=True))
    y, ty = _turn(xh * wd + bd, wd.abs() * ex + K * E * ((wd * xh).abs() + bd.abs()), pos, dims,
                  theta, interleaved, 1)
    gd, tg = _turn(g.double(), torch.zeros_like(xd), pos, dims, theta, interleaved, -1)
    gw, tw = gd * wd, tg * wd.abs()
    a0, a1 = gw.abs().mean(-1, keepdim=True), (gw * xh).abs().mean(-1, keepdim=True)
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    tdx = rstd * (K * E * (gw.abs() + a0 + xh.abs() * a1) + ex * a1
                  + xh.abs() * (gw.abs() * ex).mean(-1, keepdim=True)
                  + tw + tw.mean(-1, keepdim=True) + xh.abs() * (tw * xh.abs()).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    rows = x.numel() // d
    dw, db = (gd * xh).sum(lead), gd.sum(lead)
    wt = x.dtype if w is None else w.dtype
    bt = x.dtype if b is None else b.dtype
    tdw = (rows + K) * E * (gd * xh).abs().sum(lead) + (gd.abs() * ex + tg * xh.abs()).sum(lead)
    tdb = (rows + K) * E * gd.abs().sum(lead) + tg.sum(lead)
    return {"y": (y, ty + _half(y, x.dtype)), "dx": (dx, tdx + _half(dx, x.dtype)),
            "dw": (dw, tdw + _half(dw, wt)), "db": (db, tdb + _half(db, bt))}


def _near(got, want, what):
    v, tol = want
    o = got.detach().cpu().double()
    assert o.shape == v.shape, what
    bad = ~((o - v).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{o.numel()} off, worst "
                           f"{float(((o - v).abs() - tol).max()):.3e} beyond")


def _make(lead, heads, kv_heads, dim, dtype, wtype, seed=0, weights=NAMES[2:]):
    t = {n: (randn((*lead, h, dim), F32, seed + i) * 1.5 + 0.4).to(dtype)
         for i, (n, h) in enumerate((("q", heads), ("k", kv_heads)))}
    for i, n in enumerate(NAMES[2:]):
        t[n] = None
        if n in weights:
            t[n] = (randn((dim,), F32, seed + 5 + i) * 0.3 + (n[0] == "w")).to(wtype)
    t["gq"], t["gk"] = (randn(t[n].shape, dtype, seed + 9 + i) for i, n in enumerate("qk"))
    return t


def _call(t, **kw):
    import natten_amd

    return natten_amd.norm_rotary(*(t[n] for n in NAMES), **kw)


def _check(lead, heads, kv_heads, dim, dims, interleaved, dtype, wtype, positions=None, theta=1e4,
           eps=1e-5, seed=0, weights=NAMES[2:]):
    import natten_amd

    t = _make(lead, heads, kv_heads, dim, dtype, wtype, seed, weights)
    pos = _grid(lead) if positions is None else positions.double().expand(*lead, -1)
    d = {n: None if x is None else x.to(DEV).requires_grad_(n in NAMES) for n, x in t.items()}
    out = _call(d, positions=None if positions is None else positions.to(DEV), axis_dims=dims,
                theta=theta, interleaved=interleaved, eps=eps)
    leaves = [n for n in NAMES if d[n] is not None]
    grads = dict(zip(leaves, torch.autograd.grad(out, [d[n] for n in leaves], (d["gq"], d["gk"]))))
    dims = natten_amd.rotary_axis_dims(dim, pos.shape[-1]) if dims is None else dims
    for n, o in zip("qk", out):
        assert o.dtype == dtype and o.is_contiguous()
        want = _formula(t[n], t["w" + n], t["b" + n], t["g" + n], pos, dims, theta, interleaved, eps)
        _near(o, want["y"], f"{n}")
        _near(grads[n], want["dx"], f"d{n}")
        for w, g in (("w", "dw"), ("b", "db")):
            if t[w + n] is not None:
                assert grads[w + n].dtype == wtype
                _near(grads[w + n], want[g], f"{g} of {n}")


CASES = {
    "video, chunks of pairs": ((2, 3, 5, 7), 4, 2, 64, (16, 32, 16)),
    "video, unlike halves": ((2, 3, 5, 7), 3, 1, 64, (20, 22, 22)),
    "image of narrow heads": ((3, 9, 4), 2, 2, 32, (16, 16)),
    "image, default axes": ((1, 11, 13), 2, 1, 40, None),
    "sequence": ((2, 301), 8, 2, 128, (128,)),
    "part of the channels": ((2, 37), 5, 5, 80, (32,)),
    "odd channels": ((2, 19), 3, 2, 21, (18,)),
    "odd channels behind chunks": ((1, 33), 2, 1, 37, (16,)),
    "one pair": ((1, 5), 1, 1, 2, (2,)),
    "one token": ((1, 1), 1, 1, 64, (64,)),
    "many heads of a token": ((3, 1), 70, 9, 64, (64,)),
    "widest": ((1, 3), 2, 1, 256, (256,)),
    "widest, unlike halves": ((1, 7), 5, 2, 256, (250,)),
    "wide and odd": ((2, 2), 40, 7, 201, (118,)),
    "many tokens, unlike halves": ((2, 40, 35), 2, 1, 26, (14, 10)),
    "many tokens": ((1, 9000), 1, 1, 16, (16,)),
    "many key heads": ((2, 50), 1, 8, 48, (32,)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, BF16), (F16, F32)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", list(CASES))
def test_grid_against_the_formula(case, interleaved, dtype, wtype):
    _check(*CASES[case], interleaved, dtype, wtype)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, F32, torch.float64])
def test_positions_against_the_formula(ptype):
    g = torch.Generator().manual_seed(3)
    for shape, dims in (((4, 6, 3), (8, 12, 12)), ((6, 3), (10, 6, 16)), ((1, 6, 1), (24,)),
                        ((4, 6, 4), (4, 8, 2, 6)), ((4, 6, 2), None)):
        pos = torch.randint(-(1 << 20), 1 << 20, shape, generator=g).to(ptype)
        _check((4, 6), 3, 2, 32, dims, False, F32, F32, pos, seed=5)
    pos = torch.randint(0, 50, (2, 3, 4, 1), generator=g).to(ptype)
    _check((2, 3, 4), 2, 2, 16, (16,), True, BF16, F32, pos, theta=500.0, eps=1e-2)


@pytest.mark.gpu
@pytest.mark.parametrize("weights", [(), ("wq", "bq", "wk"), ("wk", "bk"), ("bq",), ("wq", "wk")], ids=str)
def test_missing_weights(weights):
    for dtype, wtype in ((F32, F32), (F16, F32), (BF16, BF16)):
        _check((2, 21), 3, 2, 24, (16,), False, dtype, wtype, seed=4, weights=weights)


@pytest.mark.gpu
def test_many_rows_behind_one_weight():
    """More runs of tokens than workgroups: every one of them walks."""
    _check((2, 16, 64, 24), 8, 2, 32, (8, 8, 16), False, BF16, BF16)
    _check((1, 30011), 3, 1, 20, (12,), False, F32, F32)


@pytest.mark.gpu
@pytest.mark.parametrize("dims,interleaved", [((16, 8), False), ((12, 12), False), ((12, 12), True)])
def test_views(dims, interleaved):
    packed = randn((2, 5, 6, 3, 4, 24), BF16, 1).to(DEV)
    wide = randn((2, 5, 6, 4, 30), BF16, 2).to(DEV)
    batch = randn((4, 5, 6, 4, 24), BF16, 3).to(DEV)
    cut = randn((2, 9, 6, 4, 24), BF16, 4).to(DEV)
    swapped = randn((2, 6, 5, 4, 24), BF16, 5).to(DEV)
    odd = randn((1 + 2 * 5 * 6 * 4 * 24,), BF16, 6).to(DEV)
    views = [packed[..., 0, :, :], packed[..., 1, 1:3, :], wide[..., 3:27], batch[::2], cut[:, 2:7],
             swapped.transpose(1, 2), odd[1:].view(2, 5, 6, 4, 24), batch[:1].expand(2, 5, 6, 4, 24),
             batch[:2].transpose(0, -1).contiguous().transpose(0, -1)]
    w = {n: randn((48,), BF16, 7 + i).to(DEV)[::2] for i, n in enumerate(NAMES[2:])}

    def step(q, k, gq, gk):
        d = {"q": q.detach().requires_grad_(True), "k": k.detach().requires_grad_(True),
             **{n: x.detach().requires_grad_(True) for n, x in w.items()}}
        out = _call(d, axis_dims=dims, interleaved=interleaved)
        return [*out, *torch.autograd.grad(out, [d[n] for n in NAMES], (gq, gk))]

    for q in views:
        for k in (views[1], q):
            for gq in (views[0], views[3]):
                gq = gq[..., :q.shape[-2], :]
                gk = views[5][..., :k.shape[-2], :]
                want = step(q.contiguous(), k.contiguous(), gq.contiguous(), gk.contiguous())
                for a, b in zip(step(q, k, gq, gk), want):
                    assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("twin", [False, True])
def test_missing_keys_and_gradients(twin):
    import natten_amd
    import natten_amd.autograd.fused as AF

    t = {n: x.to(DEV).requires_grad_(True) for n, x in _make((2, 7), 4, 2, 32, F32, F32).items()}
    with AF.python_autograd(twin):
        out = _call(t)
        assert ("CppNode" in out[0].grad_fn.name()) != twin
        full = torch.autograd.grad((out[0].square().sum() + out[1].sum()), [t[n] for n in NAMES])
        only = natten_amd.norm_rotary(t["q"], q_weight=t["wq"], q_bias=t["bq"])
        assert torch.equal(only, out[0])
        for part, f in ((0, lambda x: x.square().sum()), (1, lambda x: x.sum())):
            mine = [n for n in NAMES if n[-1] == "qk"[part]]
            got = torch.autograd.grad(f(_call(t)[part]), [t[n] for n in NAMES], allow_unused=True)
            for n, g, w in zip(NAMES, got, full):
                assert (g is None) if n not in mine else torch.equal(g, w), n
            for n in mine:  # one wanted alone
                d = {m: x.detach().requires_grad_(m == n) for m, x in t.items()}
                (g,) = torch.autograd.grad(f(_call(d)[part]), d[n])
                assert torch.equal(g, full[NAMES.index(n)]), n
        loss = _call(t)[0].square().sum()
        (g,) = torch.autograd.grad(loss, t["q"], retain_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable|once_differentiable"):
            torch.autograd.grad(loss, t["q"], create_graph=True)[0].sum().backward()
        # a gradient of another type, and a backward twice over the same graph
        assert torch.equal(torch.autograd.grad(loss, t["q"])[0], g)


@pytest.mark.gpu
def test_gradient_against_differences():
    """A step of h along d changes f = <y, g> by h <grad, d> up to the second
    difference, which Richardson's step takes out to h^4, and the rounding of f: 64 e
    of |y| |g| at each of four points over h."""
    import natten_amd

    t = {n: x.to(DEV) for n, x in _make((2, 4, 5), 3, 2, 24, F32, F32, 3).items()}
    t = {n: x.requires_grad_(n in NAMES) for n, x in t.items()}
    grads = torch.autograd.grad(_call(t), [t[n] for n in NAMES], (t["gq"], t["gk"]))
    for i, n in enumerate(NAMES):
        d = randn(t[n].shape, F32, 40 + i).to(DEV)

        def f(h):
            moved = {m: (x.detach() + h * d if m == n else x.detach()) for m, x in t.items()}
            out = _call(moved)
            return sum((o.double() * t[g].double()).sum().item() for o, g in zip(out, ("gq", "gk")))

        h = 2.0 ** -5
        c1, c2 = (f(h) - f(-h)) / (2 * h), (f(2 * h) - f(-2 * h)) / (4 * h)
        size = sum(float(o.detach().norm() * t[g].norm()) for o, g in zip(_call(t), ("gq", "gk")))
        noise = 2 * 64 * E * size / h + abs(c1 - c2) * 2.0 ** -3
        assert abs((4 * c1 - c2) / 3 - float((grads[i].double() * d.double()).sum())) <= noise, n


@pytest.mark.gpu
def test_no_tokens_and_special_rows():
    import natten_amd

    w = torch.ones(16, device=DEV, requires_grad=True)
    q = torch.empty(0, 5, 2, 16, device=DEV, requires_grad=True)
    out = natten_amd.norm_rotary(q, q, w, w, w, w)
    assert out[0].shape == q.shape
    gq, gw = torch.autograd.grad(out[0].sum() + out[1].sum(), (q, w))
    assert gq.shape == q.shape and not gw.any()
    assert natten_amd.norm_rotary(torch.empty(2, 0, 3, 2, 16, device=DEV)).shape == (2, 0, 3, 2, 16)
    assert natten_amd.norm_rotary(torch.empty(2, 3, 0, 16, device=DEV)).numel() == 0
    for dtype in (F32, BF16):
        for interleaved in (False, True):
            for dims in ((16,), (12,)):
                t = {n: x.to(DEV).requires_grad_(n in NAMES) for n, x in _make((1, 6), 2, 1, 20, dtype, dtype).items()}
                kw = dict(axis_dims=dims, interleaved=interleaved)

                def step():
                    out = _call(t, **kw)
                    return [*out, *torch.autograd.grad(out, (t["q"], t["k"]), (t["gq"], t["gk"]))]

                clean = step()
                with torch.no_grad():
                    t["q"][0, 2, 1, 3], t["q"][0, 4, 0, 19] = float("inf"), float("nan")
                got = step()
                keep = torch.ones(6, 2, dtype=torch.bool, device=DEV)
                keep[2, 1] = keep[4, 0] = False
                for i in (0, 2):
                    assert torch.equal(got[i][0][keep], clean[i][0][keep])
                    assert not got[i][0][~keep].isfinite().any()
                for i in (1, 3):
                    assert torch.equal(got[i], clean[i])
    # a row of equal channels is its bias, turned
    x = torch.full((1, 3, 2, 16), 0.75, device=DEV)
    b = randn((16,), F32, 1).to(DEV)
    assert torch.equal(natten_amd.norm_rotary(x, q_bias=b),
                       natten_amd.rotary(b.expand(1, 3, 2, 16).contiguous()))


@pytest.mark.gpu
def test_both_nodes_streams_and_capture():
    import natten_amd.autograd.fused as AF

    t = {n: x.to(DEV).requires_grad_(n in NAMES) for n, x in _make((2, 6, 7), 4, 2, 32, BF16, F32).items()}
    pos = torch.randint(0, 1000, (6, 7, 2), device=DEV)

    def step():
        out = _call(t, positions=pos)
        return [x.detach() for x in out] + list(
            torch.autograd.grad(out, [t[n] for n in NAMES], (t["gq"], t["gk"])))

    want = step()
    with AF.python_autograd():
        twin = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        torch.cuda.synchronize()
        graphs, helds = [], []
        for _ in range(2):  # two graphs, each with its own workspace
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=side):
                helds.append(step())
    torch.cuda.current_stream().wait_stream(side)
    for a, b, c in zip(want, twin, other):
        assert torch.equal(a, b) and torch.equal(a, c)
    for r in range(3):
        pos += 17
        with torch.no_grad():
            t["q"].copy_(randn(t["q"].shape, BF16, 30 + r))
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for held in helds:
            for a, b in zip(step(), held):
                assert torch.equal(a, b), r


@pytest.mark.gpu
def test_compiled_and_transformed():
    import natten_amd

    t = {n: x.to(DEV).requires_grad_(n in NAMES) for n, x in _make((2, 9), 3, 1, 24, F32, F32).items()}
    want = _call(t, axis_dims=(16,))
    fn = torch.compile(lambda *a: natten_amd.norm_rotary(*a, axis_dims=(16,)), backend="eager")
    for a, b in zip(fn(*(t[n] for n in NAMES)), want):
        assert torch.equal(a, b)
    for twin in (False, True):
        import natten_amd.autograd.fused as AF

        with AF.python_autograd(twin):
            for n in NAMES:
                with torch.autograd.forward_ad.dual_level():
                    d = {m: torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x)) if m == n
                         else x.detach() for m, x in t.items()}
                    with pytest.raises(NotImplementedError):
                        _call(d, axis_dims=(16,))
            with pytest.raises(RuntimeError, match="functorch"):
                torch.vmap(lambda q: natten_amd.norm_rotary(q))(t["q"].detach()[None])


def test_refusals():
    import natten_amd
    from natten_amd._core import _lib

    q, k, w = torch.randn(2, 5, 4, 16), torch.randn(2, 5, 1, 16), torch.ones(16)
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.norm_rotary(q, k, w, w, w, w)
    for args, kw, match in (
            ((torch.randn(5, 4, 16),), {}, "one to three"),
            ((q, torch.randn(2, 6, 1, 16)), {}, "batch and spatial"),
            ((q, k.half()), {}, "same dtype"),
            ((q, k), dict(axis_dims=(18,)), "rotate 18"),
            ((q, k), dict(theta=0.0), "theta"),
            ((torch.randn(1, 2, 1, 258),), {}, "up to 256"),
            ((q, k, w[:8]), {}, "q_weight must have shape"),
            ((q, k, w[None]), {}, "q_weight must have shape"),
            ((q, k, w, w, w, w[:3]), {}, "k_bias must have shape"),
            ((q, k, w.half()), {}, "or float32"),
            ((q.half(), k.half(), w, w.half()), {}, "same dtype"),
            ((q, None, w, w, w), {}, "belongs to key"),
            ((q, None), dict(k_bias=w), "belongs to key"),
            ((q, k), dict(eps=-1.0), "eps"),
            ((q, k), dict(eps=math.inf), "eps"),
            ((q, k), dict(eps=math.nan), "eps"),
            ((q, k), dict(positions=torch.zeros(2, 5, 1, requires_grad=True)), "not differentiable")):
        with pytest.raises(ValueError, match=match):
            natten_amd.norm_rotary(*args, **kw)

    lib = _lib.load()

    def params(rotary={}, **kw):
        r = _lib.NaRotaryParams(**{**dict(batch=2, heads=4, kv_heads=1, head_dim=16, dtype=2, n_axes=1,
                                          theta=1e4), **rotary})
        r.extent[0], r.extent[1], r.extent[2], r.axis_dim[0] = 1, 1, 5, 16
        return _lib.NaNormRotaryParams(**{**dict(rotary=r, weight_dtype=0, eps=1e-5), **kw})

    def fwd(p):
        return lib.na_norm_rotary_fwd(p, *([None] * 10))

    def bwd(p, dwq=None, dq=None):
        return lib.na_norm_rotary_bwd(p, *([None] * 7), dq, None, dwq, *([None] * 4), 0, None)

    assert fwd(params()) == 1 and b"non-NULL" in lib.na_last_error()
    assert bwd(params(), dq=1) == 1 and b"non-NULL" in lib.na_last_error()
    assert fwd(params(dict(batch=0))) == 0 and bwd(params()) == 0
    assert fwd(params(dict(heads=0, kv_heads=0))) == 0
    assert lib.na_norm_rotary_bwd_workspace_bytes(params()) >= 2 * 2 * 16 * 4
    for bad in (params(dict(dtype=7)), params(dict(inverse=1)), params(weight_dtype=1),
                params(eps=-1.0), params(eps=math.nan), params(eps=math.inf), params(dict(theta=-1.0))):
        assert fwd(bad) == 1 and bwd(bad, dq=1) == 1
        assert lib.na_norm_rotary_bwd_workspace_bytes(bad) == 0
    for bad in (params(dict(head_dim=258)), params(dict(head_dim=8)), params(dict(batch=1 << 30))):
        assert fwd(bad) == 2 and bwd(bad, dq=1) == 2

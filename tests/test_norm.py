"""layer_norm against its formula in float64, forward and backward: every lane
layout (lanes of a wave, four waves, sixteen waves per row), odd widths, views,
weights of either type, missing weights, empty and special rows; both
implementations of the node, streams and graph capture; and what it refuses.

Tolerances.  With e = 2^-24 (half a step of float32) and at most 32 sequential
and about 12 pairwise additions in a row's sums, K = 64 bounds the relative
error of a sum against the sum of magnitudes, and of the few operations after
it.  So |xh| is off by at most ex = K e (|xh| + rstd max|x|), y by |w| ex plus
K e (|w xh| + |b|), dx by rstd times (K e of the terms' magnitudes + what ex
moves them by), each plus half a step of the result's own type.  dw adds `rows`
terms, in chains of at most that length: (rows + K) e sum|g xh| + sum |g| ex.
"""

import pytest
import torch

from _helpers import DEV, randn

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E, K = 2.0 ** -24, 64


def _half(t, dtype):
    return t.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny


def _formula(x, w, b, g, eps):
    """Results in float64 and how far off each may be, as (value, tolerance)."""
    xd, gd = x.double(), g.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double()
    bd = torch.zeros(x.shape[-1], dtype=torch.float64) if b is None else b.double()
    mean = xd.mean(-1, keepdim=True)
    xc = xd - mean
    rstd = (xc.square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = xc * rstd
    ex = K * E * (xh.abs() + rstd * xd.abs().amax(-1, keepdim=True))
    y = xh * wd + bd
    ty = wd.abs() * ex + K * E * ((wd * xh).abs() + bd.abs()) + _half(y, x.dtype)
    gw = gd * wd
    m0, m1 = gw.mean(-1, keepdim=True), (gw * xh).mean(-1, keepdim=True)
    dx = rstd * (gw - m0 - xh * m1)
    a0, a1 = gw.abs().mean(-1, keepdim=True), (gw * xh).abs().mean(-1, keepdim=True)
    tdx = rstd * (K * E * (gw.abs() + a0 + xh.abs() * a1) + ex * a1
                  + xh.abs() * (gw.abs() * ex).mean(-1, keepdim=True)) + _half(dx, x.dtype)
    lead = tuple(range(x.dim() - 1))
    rows = x.numel() // x.shape[-1]
    dw, db = (gd * xh).sum(lead), gd.sum(lead)
    wt = x.dtype if w is None else w.dtype
    bt = x.dtype if b is None else b.dtype
    tdw = (rows + K) * E * (gd * xh).abs().sum(lead) + (gd.abs() * ex).sum(lead) + _half(dw, wt)
    tdb = (rows + K) * E * gd.abs().sum(lead) + _half(db, bt)
    return {"y": (y, ty), "dx": (dx, tdx), "dw": (dw, tdw), "db": (db, tdb)}


def _near(got, want, what):
    v, tol = want
    o = got.detach().cpu().double()
    assert o.shape == v.shape, what
    err = (o - v).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())}/{o.numel()} off; worst {float((err - tol).max()):.3e} "
                           f"beyond its tolerance")


def _case(shape, dtype, wtype, seed=0, has_w=True, has_b=True):
    x = (randn(shape, F32, seed) * 1.5 + 0.4).to(dtype)
    w = (randn(shape[-1:], F32, seed + 1) * 0.3 + 1).to(wtype) if has_w else None
    b = randn(shape[-1:], wtype, seed + 2) if has_b else None
    return x, w, b, randn(shape, dtype, seed + 3)


def _leaf(t):
    return None if t is None else t.to(DEV).requires_grad_(True)


def _step(x, w, b, g, eps=1e-5):
    import natten_amd

    ts = [_leaf(t) for t in (x, w, b)]
    y = natten_amd.layer_norm(*ts, eps)
    leaves = [t for t in ts if t is not None]
    grads = iter(torch.autograd.grad(y, leaves, g.to(DEV)))
    return {"y": y, **{n: next(grads) for n, t in zip(("dx", "dw", "db"), ts) if t is not None}}


SHAPES = [(1, 1), (3, 5), (7, 8), (2, 3, 33), (130, 64), (257, 256), (65, 513), (31, 1000),
          (9, 1001), (40, 2048), (17, 2051), (5, 4096), (3, 8200), (2, 16384), (2100, 520),
          (2050, 1999), (700, 12)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wtype", [(F32, F32), (BF16, BF16), (F16, F32), (BF16, F32)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_the_formula(shape, dtype, wtype):
    x, w, b, g = _case(shape, dtype, wtype)
    want = _formula(x, w, b, g, 1e-5)
    got = _step(x, w, b, g)
    for n in want:
        assert got[n].dtype == (dtype if n in ("y", "dx") else wtype)
        _near(got[n], want[n], f"{n} {shape} {dtype}")


@pytest.mark.gpu
@pytest.mark.parametrize("has_w,has_b", [(False, False), (True, False), (False, True)])
def test_missing_weights(has_w, has_b):
    for dtype, wtype in ((F32, F32), (F16, F32), (BF16, BF16)):
        x, w, b, g = _case((37, 72), dtype, wtype, 4, has_w, has_b)
        want, got = _formula(x, w, b, g, 1e-3), _step(x, w, b, g, 1e-3)
        assert set(got) == {"y", "dx"} | ({"dw"} if has_w else set()) | ({"db"} if has_b else set())
        for n in got:
            _near(got[n], want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(33, 96), (5, 24), (1, 3000), (1, 20), (300, 9000)], ids=str)
def test_only_some_gradients(shape):
    import natten_amd

    x, w, b, g = (t.to(DEV) for t in _case(shape, BF16, BF16, 7))
    full = _step(x, w, b, g)
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        ts = [t.detach().clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        (d,) = torch.autograd.grad(natten_amd.layer_norm(*ts), [t for t in ts if t.requires_grad], g)
        assert torch.equal(d, full[("dx", "dw", "db")[need.index(True)]])
    with torch.no_grad():
        assert torch.equal(natten_amd.layer_norm(x, w, b), full["y"])


def _views(dtype):
    packed = randn((2, 5, 7, 3, 4, 24), dtype, 1).to(DEV)
    yield "a part of a packed projection", packed[..., 1, :, :]
    yield "one head of it", packed[..., 2, 3, :]
    yield "cut channels", randn((6, 11, 40), dtype, 2).to(DEV)[..., 3:30]
    yield "an odd start", randn((1 + 9 * 31,), dtype, 3).to(DEV)[1:].view(9, 31)
    yield "every second row", randn((20, 16), dtype, 4).to(DEV)[::2]
    yield "broadcast rows", randn((1, 5, 48), dtype, 5).to(DEV).expand(4, 5, 48)
    yield "permuted rows", randn((3, 4, 5, 16), dtype, 6).to(DEV).permute(2, 0, 1, 3)
    yield "strided channels", randn((6, 16, 2), dtype, 7).to(DEV)[..., 0]
    yield "one row", randn((70, 2), dtype, 8).to(DEV)[:, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_of_inputs_and_gradients(dtype):
    import natten_amd

    inputs = list(_views(dtype))
    for name, v in inputs:
        c = v.shape[-1]
        w, b = randn((c,), dtype, 10).to(DEV), randn((c,), dtype, 11).to(DEV)
        gs = [randn(v.shape, dtype, 12).to(DEV)]
        gs += [g for _, g in inputs if g.shape == v.shape]
        gs += [torch.ones((), dtype=dtype, device=DEV).expand(v.shape),
               gs[0].transpose(0, -1).contiguous().transpose(0, -1)]
        for g in gs:
            res = []
            for x in (v.detach(), v.detach().contiguous()):
                ts = [t.detach().requires_grad_(True) for t in (x, w, b)]
                gx = g if not res else g.contiguous()
                y = natten_amd.layer_norm(*ts)
                res.append((y, *torch.autograd.grad(y, ts, gx)))
            for a, r in zip(*res):
                assert torch.equal(a, r), name
        wide = randn((2 * c,), dtype, 10).to(DEV)  # a weight with a stride
        wide[::2] = w
        assert torch.equal(natten_amd.layer_norm(v, wide[::2], b), natten_amd.layer_norm(v, w, b))


@pytest.mark.gpu
def test_views_with_different_row_orders():
    """The input one view, its gradient another, of more rows than one level."""
    import natten_amd

    x = randn((4, 6, 3, 5, 32), F32, 1).to(DEV)[:, :, 1].requires_grad_(True)   # 24 x 5 rows
    for g in (randn((4, 3, 6, 5, 32), F32, 2).to(DEV)[:, 1],                    # 4 x 30 rows
              randn((6, 4, 5, 32), F32, 3).to(DEV).transpose(0, 1), randn((4, 6, 5, 32), F32, 4).to(DEV)):
        got = torch.autograd.grad(natten_amd.layer_norm(x), x, g)[0]
        want = torch.autograd.grad(natten_amd.layer_norm(x), x, g.contiguous())[0]
        assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 64), (4, 0, 1000), (0, 9000)], ids=str)
def test_no_rows(shape):
    x, w, b, g = _case(shape, BF16, F32)
    got = _step(x, w, b, g)
    assert got["y"].shape == got["dx"].shape == shape
    assert not got["dw"].any() and not got["db"].any() and got["dw"].shape == shape[-1:]


@pytest.mark.gpu
@pytest.mark.parametrize("width", [24, 777, 5000])
def test_special_rows(width):
    """Rows that hold infinities or NaN touch no other row; equal channels give
    the bias; a mean far from zero keeps the variance."""
    x, w, b, g = _case((9, width), F32, F32, 3)
    clean = _step(x, w, b, g)
    bad = x.clone()
    bad[2, 3], bad[5, 0] = float("inf"), float("nan")
    got = _step(bad, w, b, g)
    keep = [0, 1, 3, 4, 6, 7, 8]
    assert torch.equal(got["y"][keep], clean["y"][keep])
    assert torch.equal(got["dx"][keep], clean["dx"][keep])
    assert got["y"][[2, 5]].isnan().all() and got["dw"].isnan().all()
    assert torch.equal(got["db"], clean["db"])

    x[4] = 0.75
    got = _step(x, w, b, g)
    assert torch.equal(got["y"][4].cpu(), b)
    x += 1000.0
    want, got = _formula(x, w, b, g, 1e-5), _step(x, w, b, g)
    for n in want:
        _near(got[n], want[n], n)


@pytest.mark.gpu
def test_gradients_against_differences():
    """<grad, d> against (f(x + h d) - f(x - h d)) / 2h of f = <y, g>: the
    differences' own error is h^2 times the third derivative, below 1e-4 of the
    value here, and 64 e sum|y g| / h of rounding."""
    import natten_amd

    ts = [t.to(DEV) for t in _case((40, 130), F32, F32, 11)]
    g = ts.pop()
    grads = _step(*(t.cpu() for t in ts), g.cpu())

    def f(args):
        return (natten_amd.layer_norm(*args).double() * g.double()).sum().item()

    h = 1e-2
    for i, n in enumerate(("dx", "dw", "db")):
        d = randn(ts[i].shape, F32, 20 + i).to(DEV)
        d = d / d.norm()
        up, down = [[t + s * h * d if j == i else t for j, t in enumerate(ts)] for s in (1, -1)]
        diff = (f(up) - f(down)) / (2 * h)
        exact = (grads[n].double() * d.double()).sum().item()
        noise = 64 * E * float((natten_amd.layer_norm(*ts) * g).double().norm()) / h
        assert abs(diff - exact) <= 1e-4 * float(grads[n].norm()) + noise, n


@pytest.mark.gpu
def test_both_nodes_streams_and_capture():
    import natten_amd
    import natten_amd.autograd.fused as AF

    x, w, b, g = (t.to(DEV) for t in _case((3, 50, 200), BF16, F32, 5))
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))

    def step():
        y = natten_amd.layer_norm(x, w, b)
        return [y.detach(), *torch.autograd.grad(y, (x, w, b), g)]

    want = step()
    with AF.python_autograd():
        twin = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, t, o in zip(want, twin, other):
        assert torch.equal(a, t) and torch.equal(a, o)
    for k in range(3):
        with torch.no_grad():
            x.copy_(randn(x.shape, BF16, 30 + k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, r in zip(step(), held):
            assert torch.equal(a, r), k


@pytest.mark.gpu
def test_refuses_a_second_derivative():
    import natten_amd
    import natten_amd.autograd.fused as AF

    x = randn((4, 16)).to(DEV).requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(natten_amd.layer_norm(x).square().sum(), x, create_graph=True)
    with AF.python_autograd():
        (d,) = torch.autograd.grad(natten_amd.layer_norm(x).square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            d.sum().backward()


def test_refusals():
    import natten_amd
    from natten_amd._core import _lib

    x, w = torch.randn(4, 8), torch.randn(8)
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.layer_norm(x, w, w)
    for bad in (torch.randn(()), torch.randn(3, 0), torch.randn(1, 16385)):
        with pytest.raises(ValueError, match="C from 1 to 16384"):
            natten_amd.layer_norm(bad)
    with pytest.raises(ValueError, match="weight must have shape"):
        natten_amd.layer_norm(x, torch.randn(7))
    with pytest.raises(ValueError, match="bias must have shape"):
        natten_amd.layer_norm(x, w, torch.randn(8, 1))
    with pytest.raises(ValueError, match="or float32"):
        natten_amd.layer_norm(x, w.half())
    with pytest.raises(ValueError, match="the same dtype"):
        natten_amd.layer_norm(x.half(), w, w.half())
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            natten_amd.layer_norm(x, w, eps=eps)
    with pytest.raises((TypeError, RuntimeError)):
        natten_amd.layer_norm(x.double())

    lib = _lib.load()
    p = _lib.NaNormParams(rows=4, channels=8, dtype=_lib.NA_BF16, weight_dtype=_lib.NA_F16, eps=1e-5,
                          inner=1)
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 1
    assert b"weight dtype" in lib.na_last_error()
    p.weight_dtype = _lib.NA_F32
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 1
    assert lib.na_norm_bwd(p, *([None] * 8), 0, None) == 0  # nothing wanted
    assert lib.na_norm_bwd_workspace_bytes(p) == 0  # one workgroup writes its sums itself
    p.rows = 4096
    assert lib.na_norm_bwd_workspace_bytes(p) >= 2 * 2 * 8 * 4  # two float rows a workgroup
    p.rows = 1 << 30
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 2
    p.rows, p.channels = 4, 16385
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 2
    p.channels, p.inner = 8, 0
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 1
    p.inner, p.rows = 1, 0
    assert lib.na_norm_fwd(p, None, None, None, None, None, None) == 0  # no rows

"""rotary against its formula in float64, forward and backward: pairs half an axis
apart and side by side, every unit that a row is split into, grids of one to
three axes and tensors of positions near and far, views, missing keys and
gradients, both implementations of the node, streams and graph capture; and what
it refuses.

Tolerance.  With e = 2^-24: the angle, in turns and reduced to half a turn, is
rounded to float32 once (off by at most 1.6 e in angle; its float64 parts add
less than 2^-30 at a million positions), sine and cosine add at most 2.5 e, the
two products and the sum 3 e of |u| + |v|.  So each channel is off by at most
8 e (|u| + |v|) plus half a step of its own type.
"""

import math

import pytest
import torch

from _helpers import DEV, randn

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24


def _formula(x, pos, dims, theta, interleaved, sign=1.0):
    """(value, tolerance) of x [B, *S, H, D] at pos [B, *S, axes] (float64)."""
    out = x.double().clone()
    tol = torch.zeros_like(out)
    first = 0
    for a, d in enumerate(dims):
        for i in range(d // 2):
            c0, c1 = (first + 2 * i, first + 2 * i + 1) if interleaved else (first + i, first + i + d // 2)
            angle = sign * pos[..., a, None].double() * theta ** (-2.0 * i / d)
            u, v = x[..., c0].double(), x[..., c1].double()
            out[..., c0] = u * angle.cos() - v * angle.sin()
            out[..., c1] = u * angle.sin() + v * angle.cos()
            tol[..., c0] = tol[..., c1] = 8 * E * (u.abs() + v.abs())
        first += d
    half = out.abs() * torch.finfo(x.dtype).eps / 2 + torch.finfo(x.dtype).tiny
    tol[..., :first] += half[..., :first]
    return out, tol


def _near(got, want, what):
    v, tol = want
    o = got.detach().cpu().double()
    assert o.shape == v.shape, what
    bad = ~((o - v).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())}/{o.numel()} off, worst {float((o - v).abs().max()):.3e}"


def _grid(lead):
    axes = [torch.arange(n, dtype=torch.float64) for n in lead[1:]]
    return torch.stack(torch.meshgrid(*axes, indexing="ij"), -1).expand(*lead, -1)


def _check_case(lead, heads, kv_heads, dim, dims, interleaved, dtype, positions=None, theta=1e4,
                seed=0):
    import natten_amd

    q, k = randn((*lead, heads, dim), dtype, seed), randn((*lead, kv_heads, dim), dtype, seed + 1)
    gq, gk = randn(q.shape, dtype, seed + 2), randn(k.shape, dtype, seed + 3)
    pos = _grid(lead) if positions is None else positions.double().expand(*lead, -1)
    qd, kd = (t.to(DEV).requires_grad_(True) for t in (q, k))
    oq, ok = natten_amd.rotary(qd, kd, positions=None if positions is None else positions.to(DEV),
                               axis_dims=dims, theta=theta, interleaved=interleaved)
    dq, dk = torch.autograd.grad((oq, ok), (qd, kd), (gq.to(DEV), gk.to(DEV)))
    dims = natten_amd.rotary_axis_dims(dim, pos.shape[-1]) if dims is None else dims
    for x, o, sign, n in ((q, oq, 1, "q"), (k, ok, 1, "k"), (gq, dq, -1, "dq"), (gk, dk, -1, "dk")):
        assert o.dtype == dtype and o.is_contiguous()
        _near(o, _formula(x, pos, dims, theta, interleaved, sign), n)


CASES = {
    "video, chunks of pairs": ((2, 3, 5, 7), 4, 2, 64, (16, 32, 16)),
    "video, single pairs": ((2, 3, 5, 7), 3, 1, 64, (20, 22, 22)),
    "image": ((3, 9, 4), 2, 2, 32, (16, 16)),
    "image, default axes": ((1, 11, 13), 2, 1, 40, None),
    "sequence": ((2, 301), 8, 2, 128, (128,)),
    "part of the channels": ((2, 37), 5, 5, 80, (32,)),
    "odd channels": ((2, 19), 3, 2, 21, (18,)),
    "odd channels behind chunks": ((1, 33), 2, 1, 37, (16, )),
    "one pair": ((1, 5), 1, 1, 2, (2,)),
    "one token": ((1, 1), 1, 1, 64, (64,)),
    "many heads of a token": ((3, 1), 70, 9, 64, (64,)),
    "widest": ((1, 3), 2, 1, 640, (512,)),
    "widest, unlike halves": ((1, 3), 5, 2, 1024, (510,)),
    "many wide heads, unlike halves": ((2, 2), 40, 7, 300, (118,)),
    "many tokens, unlike halves": ((2, 40, 35), 2, 1, 26, (14, 10)),
    "many tokens": ((1, 5000), 1, 1, 16, (16,)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("case", list(CASES))
def test_grid_against_the_formula(case, interleaved, dtype):
    _check_case(*CASES[case], interleaved, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, F32, torch.float64])
@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_against_the_formula(ptype, interleaved):
    g = torch.Generator().manual_seed(3)
    for shape, dims in (((4, 6, 3), (8, 12, 12)), ((6, 3), (10, 6, 16)), ((1, 6, 1), (24,)),
                        ((4, 6, 4), (4, 8, 2, 6)), ((4, 6, 2), None)):
        pos = torch.randint(-(1 << 20), 1 << 20, shape, generator=g).to(ptype)
        if ptype.is_floating_point:
            pos = pos + 0.25  # exact in float32 up to 2^21
        _check_case((4, 6), 3, 2, 32, dims, interleaved, F32, pos, seed=5)
    # one position per token of an image
    pos = torch.randint(0, 50, (2, 3, 4, 1), generator=g).to(ptype)
    _check_case((2, 3, 4), 2, 2, 16, (16,), interleaved, BF16, pos, theta=500.0)


@pytest.mark.gpu
def test_far_positions_keep_neighbours_apart():
    """At a million tokens a float32 angle cannot tell a position from the next."""
    pos = torch.tensor([[[1 << 20], [(1 << 20) + 1], [(1 << 24) + 3], [0]]])
    _check_case((1, 4), 2, 1, 64, (64,), False, F32, pos)


@pytest.mark.gpu
@pytest.mark.parametrize("dims,interleaved", [((16, 8), False), ((12, 12), False), ((12, 12), True)])
def test_views(dims, interleaved):
    import natten_amd

    def both(q, k):
        return natten_amd.rotary(q, k, axis_dims=dims, interleaved=interleaved)

    packed = randn((2, 5, 6, 3, 4, 24), BF16, 1).to(DEV)
    wide = randn((2, 5, 6, 4, 30), BF16, 2).to(DEV)
    batch = randn((4, 5, 6, 4, 24), BF16, 3).to(DEV)
    cut = randn((2, 9, 6, 4, 24), BF16, 4).to(DEV)
    swapped = randn((2, 6, 5, 4, 24), BF16, 5).to(DEV)
    odd = randn((1 + 2 * 5 * 6 * 4 * 24,), BF16, 6).to(DEV)
    views = [packed[..., 0, :, :], packed[..., 1, 1:3, :], wide[..., 3:27], batch[::2], cut[:, 2:7],
             swapped.transpose(1, 2), odd[1:].view(2, 5, 6, 4, 24), batch[:1].expand(2, 5, 6, 4, 24),
             batch[:2].transpose(0, -1).contiguous().transpose(0, -1),
             batch[:2, :, :, :1].expand(2, 5, 6, 4, 24)]
    for q in views:
        for k in (views[1], q):
            a, b = both(q, k), both(q.contiguous(), k.contiguous())
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q = views[0].detach().requires_grad_(True)
    for g in (v for v in views if v.shape == q.shape):
        out = natten_amd.rotary(q, axis_dims=dims, interleaved=interleaved)
        d1 = torch.autograd.grad(out, q, g, retain_graph=True)[0]
        assert torch.equal(d1, torch.autograd.grad(out, q, g.contiguous())[0])


@pytest.mark.gpu
def test_missing_keys_and_gradients():
    import natten_amd
    import natten_amd.autograd.fused as AF

    q, k = (randn((2, 7, h, 32), F32, h).to(DEV).requires_grad_(True) for h in (4, 2))
    oq, ok = natten_amd.rotary(q, k)
    assert torch.equal(natten_amd.rotary(q), oq)
    dq, dk = torch.autograd.grad((oq.square().sum() + ok.sum()), (q, k))
    for twin in (False, True):
        with AF.python_autograd(twin):
            a, b = natten_amd.rotary(q, k)
            assert torch.equal(torch.autograd.grad(a.square().sum(), q)[0], dq)
            a, b = natten_amd.rotary(q, k)
            assert torch.equal(torch.autograd.grad(b.sum(), k)[0], dk)
            a, b = natten_amd.rotary(q.detach(), k)
            assert torch.equal(torch.autograd.grad(b.sum(), k)[0], dk)
            # the map is linear: its second derivative along a direction is exact
            (g,) = torch.autograd.grad(natten_amd.rotary(q).pow(3).sum(), q, create_graph=True)
            (h,) = torch.autograd.grad(g.sum(), q)
    x = natten_amd.rotary(q).detach()
    ones = torch.ones_like(x)
    turned = natten_amd.rotary(ones)
    want = torch.ops.natten_amd.na_rotary(6 * x * turned, None, None, [32], 1e4, False, True,
                                          torch.cuda.current_stream().cuda_stream)[0]
    assert torch.allclose(h, want, rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
def test_gradient_against_differences():
    """The map is linear: (f(x + h d) - f(x - h d)) / 2h is its gradient along d up
    to the rounding of f, 16 e |x| |g| / h."""
    import natten_amd

    x, g, d = (randn((2, 4, 5, 3, 24), F32, s).to(DEV) for s in (1, 2, 3))
    x.requires_grad_(True)
    (dx,) = torch.autograd.grad(natten_amd.rotary(x), x, g)

    def f(t):
        return (natten_amd.rotary(t.detach()).double() * g.double()).sum().item()

    h = 0.5
    diff = (f(x + h * d) - f(x - h * d)) / (2 * h)
    noise = 16 * E * float(x.detach().norm() + d.norm()) * float(g.norm()) / h
    assert abs(diff - float((dx.double() * d.double()).sum())) <= noise


@pytest.mark.gpu
def test_no_tokens_and_special_values():
    import natten_amd

    q = torch.empty(0, 5, 2, 16, device=DEV, requires_grad=True)
    out = natten_amd.rotary(q)
    assert out.shape == q.shape and torch.autograd.grad(out.sum(), q)[0].shape == q.shape
    assert natten_amd.rotary(torch.empty(2, 0, 3, 2, 16, device=DEV)).shape == (2, 0, 3, 2, 16)
    assert natten_amd.rotary(torch.empty(2, 3, 0, 16, device=DEV)).numel() == 0
    for interleaved in (False, True):
        for dims in ((16,), (12,)):
            x = randn((1, 6, 2, 20), F32, 1).to(DEV)
            clean = natten_amd.rotary(x, axis_dims=dims, interleaved=interleaved)
            x[0, 2, 1, 3], x[0, 4, 0, 19] = float("inf"), float("nan")
            got = natten_amd.rotary(x, axis_dims=dims, interleaved=interleaved)
            keep = torch.ones(6, 2, dtype=torch.bool, device=DEV)
            keep[2, 1] = keep[4, 0] = False
            assert torch.equal(got[0][keep], clean[0][keep])
            assert torch.equal(got[0, 4, 0, :19], clean[0, 4, 0, :19]) and got[0, 4, 0, 19].isnan()


@pytest.mark.gpu
def test_both_nodes_streams_and_capture():
    import natten_amd
    import natten_amd.autograd.fused as AF

    q, k = (randn((2, 6, 7, h, 32), BF16, h).to(DEV).requires_grad_(True) for h in (4, 2))
    gq, gk = (randn(t.shape, BF16, 9).to(DEV) for t in (q, k))
    pos = torch.randint(0, 1000, (6, 7, 2), device=DEV)

    def step():
        out = natten_amd.rotary(q, k, positions=pos)
        return [t.detach() for t in out] + list(torch.autograd.grad(out, (q, k), (gq, gk)))

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
    for r in range(3):
        pos += 17
        with torch.no_grad():
            q.copy_(randn(q.shape, BF16, 30 + r))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, t in zip(step(), held):
            assert torch.equal(a, t), r


def test_axis_dims():
    import natten_amd

    assert natten_amd.rotary_axis_dims(64, 3) == (20, 22, 22)
    assert natten_amd.rotary_axis_dims(64, 2) == (32, 32)
    assert natten_amd.rotary_axis_dims(6, 3) == (2, 2, 2)
    for d, n in ((63, 1), (4, 3), (8, 0)):
        with pytest.raises(ValueError, match="axes"):
            natten_amd.rotary_axis_dims(d, n)


def test_refusals():
    import natten_amd
    from natten_amd._core import _lib

    q, k = torch.randn(2, 5, 4, 16), torch.randn(2, 5, 1, 16)
    with pytest.raises(RuntimeError, match="HIP"):
        natten_amd.rotary(q, k)
    for args, match in (
            ((torch.randn(5, 4, 16),), "one to three"),
            ((q, torch.randn(2, 6, 1, 16)), "batch and spatial"),
            ((q, torch.randn(2, 5, 1, 8)), "Head dim"),
            ((q, k.half()), "same dtype"),
            ((q, k, torch.zeros(2, 4, 1)), "positions must be"),
            ((q, k, torch.zeros(5)), "positions must be"),
            ((q, k, torch.zeros(2, 5, 5)), "1 to 4 axes"),
            ((q, k, torch.zeros(2, 5, 1).half()), "positions must be int32"),
            ((q, k, torch.zeros(2, 5, 1, requires_grad=True)), "not differentiable"),
            ((q, k, None, (8, 8)), "one entry per axis"),
            ((q, k, None, (7,)), "positive even ints"),
            ((q, k, None, (0,)), "positive even ints"),
            ((q, k, None, (8.0,)), "positive even ints"),
            ((q, k, None, (18,)), "rotate 18 channels"),
            ((torch.randn(1, 2, 1, 600), None, None, (514,)), "at most 512"),
            ((torch.randn(1, 2, 1, 15),), "must be even"),
            ((torch.randn(1, 2, 1, 1026),), "up to 1024"),
            ((q, k, None, None, 0.0), "theta"),
            ((q, k, None, None, float("inf")), "theta")):
        with pytest.raises(ValueError, match=match):
            natten_amd.rotary(*args)
    with pytest.raises((TypeError, RuntimeError)):
        natten_amd.rotary(q.double())

    lib = _lib.load()

    def params(**kw):
        p = _lib.NaRotaryParams(batch=2, heads=4, kv_heads=1, head_dim=16, dtype=0, n_axes=1,
                                theta=1e4)
        p.extent[0], p.extent[1], p.extent[2], p.axis_dim[0] = 1, 1, 5, 16
        for n, v in kw.items():
            setattr(p, n, v)
        return p

    def rc(p):
        return lib.na_rotary(p, *([None] * 6))

    assert rc(params()) == 1 and b"non-NULL" in lib.na_last_error()
    assert rc(params(batch=0)) == 0 and rc(params(heads=0, kv_heads=0)) == 0
    for bad in (dict(dtype=7), dict(n_axes=0), dict(n_axes=5), dict(theta=-1.0), dict(pos_type=9),
                dict(n_axes=4), dict(theta=math.inf), dict(heads=-1)):
        assert rc(params(**bad)) == 1, bad
    assert rc(params(head_dim=8)) == 2
    assert rc(params(batch=1 << 30)) == 2
    assert rc(params(heads=1 << 20)) == 2
    p = params()
    p.axis_dim[0] = 3
    assert rc(p) == 1

"""Calls at the edges of what the layer norm, rotary positions and shared-prefix
attention document: the widest windows of the C ABI; lengths on the host;
probabilities far below a row's largest; forward-mode tangents and torch.func
transforms, which none of them takes; layers of heads that rotary does not take;
layers pickled before they had norms and positions; second derivatives of rotary
positions; rows of equal channels."""

import io
import math

import pytest
import torch

from _helpers import DEV, randn
from test_prefix import _make, _near, _reference

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24


def _prefix_c(t, window):
    """prefix_attention through the C ABI, contiguous inputs."""
    from natten_amd._core import _lib

    d = {n: x.to(DEV) for n, x in t.items() if isinstance(x, torch.Tensor)}
    B, L, H, D = t["q"].shape
    N, Hk = t["pk"].shape[:2]
    S = t["k"].shape[1]
    p = _lib.NaPrefixParams(batch=B, tokens=L, heads=H, kv_heads=Hk, head_dim=D,
                            dtype=_lib.dtype_code(t["q"].dtype), prefix=N, capacity=S, window=window,
                            scale=D ** -0.5, seq_lens=d["lens"].data_ptr())
    p.q_stride[:] = (L * H * D, H * D, D)
    p.prefix_k_stride[:] = p.prefix_v_stride[:] = (Hk * D, D)
    p.k_stride[:] = p.v_stride[:] = (S * Hk * D, Hk * D, D)
    lib = _lib.load()
    out = torch.empty_like(d["q"])
    lse = torch.empty(B, L, H, device=DEV)
    ws = torch.empty(int(lib.na_prefix_workspace_bytes(p)), dtype=torch.uint8, device=DEV)
    _lib.check(lib.na_prefix_fwd(p, *(d[n].data_ptr() for n in ("q", "pk", "pv", "k", "v")),
                                 out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws.numel(),
                                 _lib.stream_of(d["q"])), "na_prefix_fwd")
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tokens,heads", [(4, 2), (16, 4), (70, 4)])
def test_the_widest_windows_are_none(tokens, heads, dtype):
    """Samples that hold fewer own tokens than there are new ones, under windows up
    to the largest int32: every row sees all its own tokens."""
    t = _make((4, tokens, heads, 2, 64, 40, 300, [300, 4, 0, 1], None), dtype, 3)
    want_out, want_lse = _reference(t)
    for window in (0, 1 << 30, (1 << 30) + 1, (1 << 31) - 1):
        out, lse = _prefix_c(t, window)
        _near(out, want_out, f"window {window} out")
        _near(lse, want_lse, f"window {window} lse")


def _calls(device):
    """Each operator as a function of its tensors, and the tensors."""
    import natten_amd

    def r(*shape):
        return randn(shape, F32, len(shape)).to(device)

    return {
        "layer_norm": (natten_amd.layer_norm, [r(6, 16), r(16), r(16)]),
        "rotary": (lambda q, k: torch.cat([t.flatten() for t in natten_amd.rotary(q, k)]),
                   [r(2, 5, 4, 16), r(2, 5, 1, 16)]),
        "prefix": (natten_amd.prefix_attention, [r(2, 1, 4, 16), r(5, 2, 16), r(5, 2, 16), r(2, 7, 2, 16),
                                                 r(2, 7, 2, 16)]),
    }


def _dual(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.gpu
@pytest.mark.parametrize("twin", [False, True])
@pytest.mark.parametrize("name", ["layer_norm", "rotary", "prefix"])
def test_tangents_and_transforms_are_refused(name, twin):
    """No result without the tangent that the caller asks for, whichever input has
    one; without a tangent a forward-mode level changes nothing."""
    import natten_amd.autograd.fused as AF

    fn, ts = _calls(DEV)[name]
    with AF.python_autograd(twin):
        want = fn(*ts)
        for no_grad in (False, True):
            for i in range(len(ts)):
                with torch.set_grad_enabled(not no_grad), torch.autograd.forward_ad.dual_level():
                    with pytest.raises(NotImplementedError):
                        fn(*(_dual(t) if j == i else t for j, t in enumerate(ts)))
                    assert torch.equal(fn(*ts), want)
        with pytest.raises(RuntimeError, match="functorch"):
            torch.func.jvp(fn, tuple(ts), tuple(torch.ones_like(t) for t in ts))
        with pytest.raises(RuntimeError, match="functorch|no backward"):
            torch.func.grad(lambda *a: fn(*a).sum())(*ts)
        with pytest.raises(RuntimeError, match="functorch"):
            torch.vmap(fn)(*(t[None].repeat(2, *[1] * t.dim()) for t in ts))


def test_the_prefix_call_outside_the_operator_keeps_no_primal(monkeypatch):
    """The Python path, its kernels replaced by a copy of the query."""
    import natten_amd
    from natten_amd._core import hip

    monkeypatch.setattr(hip, "prefix_forward", lambda q, *rest: (q.clone(), None))
    _, (q, pk, pv, k, v) = _calls("cpu")["prefix"]
    with torch.autograd.forward_ad.dual_level():
        assert torch.equal(natten_amd.prefix_attention(q, pk, pv, k, v), q)
        for args in ((_dual(q), pk, pv, k, v), (q, _dual(pk), pv, k, v), (q, pk, pv, k, _dual(v))):
            with pytest.raises(NotImplementedError):
                natten_amd.prefix_attention(*args)
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.jvp(lambda q: natten_amd.prefix_attention(q, pk, pv, k, v), (q,), (q,))


@pytest.mark.parametrize("at", range(5))
def test_the_operators_refuse_tangents(at):
    """Direct calls of the registered operators."""
    from natten_amd._core import _lib

    _lib.load()
    ops = torch.ops.natten_amd
    calls = _calls("cpu")
    with torch.autograd.forward_ad.dual_level():
        ts = [_dual(t) if i == at else t for i, t in enumerate(calls["prefix"][1])]
        with pytest.raises(RuntimeError, match="no backward"):
            ops.na_prefix(*ts, None, 0, 0.25, False, 0)


@pytest.mark.gpu
def test_lengths_on_the_host_are_not_kept():
    """Every step of a generation has other lengths: a copy of each, kept for calls to
    come, would stay for the life of the process and crowd out the copies of lengths
    that do come again."""
    import natten_amd
    from natten_amd.autograd import fused

    t = {n: x.to(DEV) for n, x in _make((2, 1, 4, 2, 16, 5, 40, [0], None), F32).items()
         if isinstance(x, torch.Tensor)}

    def step(lens):
        return natten_amd.prefix_attention(t["q"], t["pk"], t["pv"], t["k"], t["v"], seq_lens=lens)

    before = dict(fused._extents_cache)
    for n in range(1, 30):
        lens = torch.tensor([n, 40 - n], dtype=(torch.int32, torch.int64)[n % 2])
        assert torch.equal(step(lens), step(lens.to(DEV)))
    assert fused._extents_cache == before

    lens = torch.tensor([7, 9])
    want = step(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_device = lens.to(DEV)
        step(on_device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            with pytest.raises(RuntimeError, match="on the host"):
                step(lens)
            held = step(on_device)  # the capture goes on
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(held, want) and torch.equal(step(lens), want)


SMALL = {  # B, tokens, heads, kv heads, dim, prefix, own capacity, lengths
    "narrow": (2, 1, 4, 2, 64, 320, 200, [200, 33]),
    "narrow, tokens": (2, 3, 4, 1, 32, 96, 300, [300, 70]),
    "wide of 64": (8, 1, 8, 2, 128, 320, 130, [130, 0, 64]),
    "wide of 128": (2, 70, 4, 1, 32, 160, 300, [300, 75]),
    "wide of 128, 80 wide": (3, 40, 4, 1, 80, 352, 100, [100, 41]),
    "256 wide": (5, 3, 8, 1, 256, 96, 64, [64, 7]),
    "eight waves": (40, 1, 8, 2, 128, 640, 32, [32, 0]),
    "eight waves, tokens": (3, 100, 6, 2, 128, 704, 130, [130, 101]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("case", list(SMALL))
def test_probabilities_far_below_the_largest(case, dtype):
    """Every 32nd key scores 18 and holds zeros, the others score 0 and hold 1024: a
    row of h and n of them is 1024 n e^-18 / (h + n e^-18), all of it probabilities of
    2^-26 of the largest.

    A score is off by d = 2^-24 (18 D + 2 * 18 + 16 + keys), with the sums over the keys
    (as in test_prefix); 16-bit types round a probability by u = eps / 2 of it.  fp16
    below 2^-14 rounds by 2^-25: with the largest at 2^7 at least, the n = 31 h (and up to
    31 more where a sequence ends) move a row by 1024 (n / h) 2^-32."""
    import natten_amd

    B, L, H, Hk, D, N, S, lens = SMALL[case]
    lens = torch.tensor([lens[b % len(lens)] for b in range(B)], dtype=torch.int32)
    q, pk, k = torch.zeros(B, L, H, D), torch.zeros(N, Hk, D), torch.zeros(B, S, Hk, D)
    q[..., 0], pk[::32, :, 0], k[:, ::32, :, 0] = 1.0, 18.0, 18.0
    pv, v = torch.full_like(pk, 1024.0), torch.full_like(k, 1024.0)
    pv[::32], v[:, ::32] = 0.0, 0.0
    out, lse = natten_amd.prefix_attention(*(t.to(DEV, dtype) for t in (q, pk, pv, k, v)),
                                           lens.to(DEV), scale=1.0, return_lse=True)
    out, lse = out.cpu().double(), lse.cpu().double()
    u, fi = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2, torch.finfo(dtype)
    for b in range(B):
        for j in range(L):
            own = max(0, int(lens[b]) - L + j + 1)
            h = N // 32 + -(-own // 32)
            n = N + own - h
            tail = n * math.exp(-18.0)
            want, d = 1024 * tail / (h + tail), E * (18 * D + 52 + N + own)
            tol = (u + 4 * d + fi.eps / 2) * want + fi.tiny
            if dtype == F16:
                tol += 1024 * n / h * 2.0 ** -32
            assert ((out[b, j] - want).abs() <= tol).all(), (b, j, out[b, j].min(), out[b, j].max(), want)
            ref = 18.0 + math.log(h + tail)
            assert ((lse[b, j] - ref).abs() <= 4 * d + 4 * E * (1 + ref)).all(), (b, j)


def test_layers_refuse_what_rotary_refuses():
    """At construction, not at the first call: more rotated channels than a launch's
    table holds, or heads too wide, also where the layer shares the channels out."""
    from natten_amd import nn

    for cls, dim, rotary in ((nn.NeighborhoodAttention1D, 1024, True), (nn.NeighborhoodAttention1D, 514, (514,)),
                             (nn.NeighborhoodAttention2D, 520, (260, 254)),
                             (nn.NeighborhoodAttention1D, 1026, (64,))):
        with pytest.raises(ValueError, match="rotary must be"):
            cls(dim, 1, 3, rotary=rotary)
    assert nn.NeighborhoodAttention1D(1024, 1, 3, rotary=(512,)).rotary_dims == (512,)
    assert nn.NeighborhoodAttention1D(1024, 2, 3, rotary=True).rotary_dims == (512,)
    for theta in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError, match="rotary_theta"):
            nn.NeighborhoodAttention1D(32, 2, 3, rotary=True, rotary_theta=theta)
    for eps in (-1e-5, math.nan):
        with pytest.raises(ValueError, match="eps"):
            nn.LayerNorm(8, eps)


def _pickled(m):
    f = io.BytesIO()
    torch.save(m, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


def _plain_and_older():
    from natten_amd import nn

    m = nn.NeighborhoodAttention2D(32, 2, 3)
    older = nn.NeighborhoodAttention2D(32, 2, 3)
    older.load_state_dict(m.state_dict())
    for n in ("q_norm", "k_norm", "rotary_dims", "rotary_theta"):
        del older.__dict__[n]
    return m, _pickled(older)


def test_layers_pickled_before_they_had_norms_and_positions():
    m, older = _plain_and_older()
    assert older.q_norm is None and older.k_norm is None and older.rotary_dims is None
    with pytest.raises(RuntimeError, match="HIP"):
        older(torch.randn(1, 4, 4, 32))
    from natten_amd import nn

    full = nn.NeighborhoodAttention2D(32, 2, 3, qk_norm=True, rotary=True, rotary_theta=7.0)
    back = _pickled(full)
    assert back.rotary_dims == (8, 8) and back.rotary_theta == 7.0
    assert torch.equal(back.q_norm.weight, full.q_norm.weight)


@pytest.mark.gpu
def test_layers_pickled_before_run_as_plain_ones():
    m, older = (t.to(DEV) for t in _plain_and_older())
    x = randn((2, 9, 7, 32), F32, 1).to(DEV)
    assert torch.equal(older(x), m(x))


@pytest.mark.gpu
@pytest.mark.parametrize("twin", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_second_derivatives_of_rotary(interleaved, twin):
    """f = sum oq^2 ok with (oq, ok) the rotated (q, k), and the gradient of
    <df/dq, u> + <df/dk, w>, which is R^T(2 ok Ru + 2 oq Rw) and R^T(2 oq Ru), against
    float64 matrices.  Every rotation is two products and a sum of terms of at most b
    and of a table off by 2 e; with the two factors that they meet, 64 e times the
    largest term bounds the chain of four."""
    import natten_amd
    import natten_amd.autograd.fused as AF

    q, k, u, w = (randn((2, 7, 3, 16), F32, s).to(DEV) for s in range(4))
    q.requires_grad_(True), k.requires_grad_(True)
    with AF.python_autograd(twin):
        oq, ok = natten_amd.rotary(q, k, axis_dims=(12,), interleaved=interleaved)
        assert ("CppNode" in oq.grad_fn.name()) != twin
        gq, gk = torch.autograd.grad((oq.square() * ok).sum(), (q, k), create_graph=True)
        hq, hk = torch.autograd.grad((gq * u).sum() + (gk * w).sum(), (q, k))

    rot = torch.eye(16, dtype=torch.float64).repeat(7, 1, 1)  # [token, out, in]
    for t in range(7):
        for i in range(6):
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 6)
            angle = t * 10000.0 ** (-2 * i / 12)
            rot[t, a, a] = rot[t, b, b] = math.cos(angle)
            rot[t, a, b], rot[t, b, a] = -math.sin(angle), math.sin(angle)

    def turn(x):
        return (rot[None, :, None] @ x.unsqueeze(-1)).squeeze(-1)

    def back(x):
        return (rot.transpose(1, 2)[None, :, None] @ x.unsqueeze(-1)).squeeze(-1)

    q, k, u, w = (turn(t.detach().cpu().double()) for t in (q, k, u, w))
    largest = 4 * max(float(t.abs().max()) for t in (q, k)) * max(float(t.abs().max()) for t in (u, w))
    for got, want in ((gq, back(2 * q * k)), (gk, back(q * q)),
                      (hq, back(2 * k * u + 2 * q * w)), (hk, back(2 * q * u))):
        assert (got.detach().cpu().double() - want).abs().max() <= 64 * E * largest


@pytest.mark.gpu
@pytest.mark.parametrize("width", [24, 100, 200, 500, 777, 5000, 16384])
def test_rows_of_equal_channels(width):
    """The sum of equal channels rounds, so their mean is off by up to K e of it (K = 64,
    as in test_norm) and the rows by that over sqrt(eps): no row leaves its bias by more,
    and a value whose sums are exact not at all."""
    import natten_amd

    values = torch.tensor([0.1, 1.7, 3.14159, -1e-3, 12345.678, 0.75, 0.0])
    x = values[:, None].expand(-1, width).contiguous().to(DEV)
    w, b = (randn((width,), F32, s).to(DEV) for s in (1, 2))
    for eps in (1e-5, 1e-2):
        y = natten_amd.layer_norm(x, w, b, eps)
        off = (y - b).abs().double() / w.abs().double()
        bound = (64 * E * values.double().abs() / math.sqrt(eps))[:, None].to(DEV)
        assert (off <= bound * (1 + 2 ** -10) + E * (y.abs() + b.abs()) / w.abs()).all()
        assert torch.equal(y[-2:], b.expand(2, -1))

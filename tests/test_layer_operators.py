"""The layer norm, rotary positions and shared-prefix attention together, as a
model uses them: layers with normalised and rotated queries and keys against a
float64 composition, their gradients and graph capture; and a text generated one
token at a time against the same layers over the whole sequence."""

import pytest
import torch

from _helpers import DEV, randn
from oracle import na as O

F32, BF16 = torch.float32, torch.bfloat16


def _layer(rank, dtype=F32, **kw):
    from natten_amd import nn

    torch.manual_seed(3)
    m = getattr(nn, f"NeighborhoodAttention{rank}D")(**kw)
    with torch.no_grad():
        for p in m.parameters():
            p.add_(0.1 * torch.randn(p.shape))
    return m.to(dtype)


def _turn(x, dims, theta):
    axes = [torch.arange(n, dtype=torch.float64) for n in x.shape[1:-2]]
    pos = torch.stack(torch.meshgrid(*axes, indexing="ij"), -1)
    out, first = [], 0
    for a, d in enumerate(dims):
        rate = theta ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        angle = (pos[..., a, None] * rate).unsqueeze(-2)
        u, v = x[..., first:first + d // 2], x[..., first + d // 2:first + d]
        out += [u * angle.cos() - v * angle.sin(), u * angle.sin() + v * angle.cos()]
        first += d
    return torch.cat(out + [x[..., first:]], -1)


def _reference(m, x, p):
    """The layer in float64 on the CPU; ``p``: its parameters by name."""
    lead, h, hk, d = x.shape[:-1], m.num_heads, m.num_kv_heads, m.head_dim
    if hk == h:
        q, k, v = torch.nn.functional.linear(x, p["qkv.weight"], p["qkv.bias"]).reshape(
            *lead, 3, h, d).unbind(-3)
    else:
        q = torch.nn.functional.linear(x, p["q_proj.weight"], p["q_proj.bias"]).reshape(*lead, h, d)
        k, v = torch.nn.functional.linear(x, p["kv_proj.weight"], p["kv_proj.bias"]).reshape(
            *lead, 2, hk, d).unbind(-3)
    if m.q_norm is not None:
        q = torch.nn.functional.layer_norm(q, (d,), p["q_norm.weight"], p["q_norm.bias"], 1e-5)
        k = torch.nn.functional.layer_norm(k, (d,), p["k_norm.weight"], p["k_norm.bias"], 1e-5)
    if m.rotary_dims is not None:
        q, k = (_turn(t, m.rotary_dims, m.rotary_theta) for t in (q, k))
    k, v = (t.repeat_interleave(h // hk, -2) for t in (k, v))
    out = O.na_forward(q, k, v, m.kernel_size, m.stride, m.dilation, m.is_causal, m.scale)
    return torch.nn.functional.linear(out.reshape(*out.shape[:-2], -1), p["proj.weight"], p["proj.bias"])


LAYERS = {
    "1d causal": (1, (2, 40, 32), dict(embed_dim=32, num_heads=2, kernel_size=9, is_causal=True,
                                       qk_norm=True, rotary=True)),
    "2d": (2, (2, 9, 11, 48), dict(embed_dim=48, num_heads=2, kernel_size=5, qk_norm=True,
                                   rotary=(12, 8), rotary_theta=100.0)),
    "2d strided gqa": (2, (1, 12, 10, 64), dict(embed_dim=64, num_heads=4, num_kv_heads=2, kernel_size=3,
                                               stride=2, qk_norm=True, rotary=True)),
    "3d rotary only": (3, (1, 4, 6, 5, 40), dict(embed_dim=40, num_heads=2, kernel_size=3, rotary=True)),
    "2d norm only": (2, (1, 8, 8, 32), dict(embed_dim=32, num_heads=4, kernel_size=3, qk_norm=True)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(LAYERS))
def test_layers_against_float64(case):
    """float32: the projections' and attention's sums of at most 100 terms of order
    one keep every value within 2e-4 of its own or of the tensor's largest."""
    rank, shape, kw = LAYERS[case]
    m = _layer(rank, **kw)
    x = randn(shape, F32, 1)
    p = {n: t.detach().double().requires_grad_(True) for n, t in m.named_parameters()}
    xr = x.double().requires_grad_(True)
    want = _reference(m, xr, p)
    g = randn(want.shape, F32, 2)
    wants = torch.autograd.grad(want, [xr, *p.values()], g.double())
    m = m.to(DEV)
    xd = x.to(DEV).requires_grad_(True)
    out = m(xd)
    grads = torch.autograd.grad(out, [xd, *m.parameters()], g.to(DEV))
    for n, a, b in zip(["out", "x", *p], [out, *grads], [want, *wants]):
        a, b = a.detach().cpu().double(), b.detach()
        assert a.shape == b.shape
        assert (a - b).abs().max() <= 2e-4 * max(1.0, float(b.abs().max())), n


@pytest.mark.gpu
def test_layer_in_16_bits_and_capture():
    m = _layer(2, BF16, embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True).to(DEV)
    ref = _layer(2, embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True).to(DEV)
    ref.load_state_dict(m.state_dict())
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    g = randn(x.shape, BF16, 2).to(DEV)

    def step(m=m, x=x, g=g):
        out = m(x)
        return [out.detach(), *torch.autograd.grad(out, list(m.parameters()), g)]

    want = step()
    # each of the layer's seven stages rounds its result by 2^-8 of it at most
    for a, b in zip(want, step(ref, x.float(), g.float())):
        assert (a.float() - b).norm() <= 7 * 2 ** -8 * b.norm() + 1e-6
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for r in range(3):
        x.copy_(randn(x.shape, BF16, 10 + r))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(), held):
            assert torch.equal(a, b), r


@pytest.mark.gpu
@pytest.mark.parametrize("hk", [4, 2])
def test_generation_token_by_token(hk):
    """Three texts behind one shared prefix of tokens, through two layers: caches
    filled by a chunk of a prompt, then token by token, against the layers over the
    whole sequences with the prefix as additional tokens."""
    import natten_amd

    B, T, N, C, H, K = 3, 37, 21, 64, 4, 16
    layers = [_layer(1, embed_dim=C, num_heads=H, num_kv_heads=hk, kernel_size=K, is_causal=True,
                     qk_norm=True, rotary=True).to(DEV) for _ in range(2)]
    norms = [natten_amd.nn.LayerNorm(C).to(DEV) for _ in range(2)]
    x = randn((B, T, C), F32, 1).to(DEV)
    shared = [[randn((N, hk, C // H), F32, 10 * i + s).to(DEV) for s in (2, 3)] for i in range(2)]

    def project(m, h, first):
        pos = torch.arange(first, first + h.shape[1], device=DEV).view(-1, 1)
        if hk == H:
            q, k, v = m._split_qkv(m.qkv(h))
        else:
            q = m.q_proj(h).view(*h.shape[:2], H, C // H)
            k, v = m.kv_proj(h).view(*h.shape[:2], 2, hk, C // H).unbind(-3)
        q, k = natten_amd.rotary(m.q_norm(q), m.k_norm(k), positions=pos, axis_dims=m.rotary_dims)
        return q, k, v

    with torch.no_grad():
        want = x
        for m, nm, (pk, pv) in zip(layers, norms, shared):
            q, k, v = project(m, nm(want), 0)
            o = natten_amd.na1d(q, k, v, kernel_size=K, is_causal=True,
                                additional_keys=pk.expand(B, -1, -1, -1),
                                additional_values=pv.expand(B, -1, -1, -1))
            want = want + m.proj(o.flatten(-2))
        caches = [[torch.full((B, T + 5, hk, C // H), float("nan"), device=DEV) for _ in "kv"]
                  for _ in range(2)]
        got, at = [], 0
        for n in (12, 1, 7, *([1] * (T - 20))):
            h = x[:, at:at + n]
            lens = torch.full((B,), at + n, dtype=torch.int32, device=DEV)
            for m, nm, (pk, pv), (ck, cv) in zip(layers, norms, shared, caches):
                q, k, v = project(m, nm(h), at)
                ck[:, at:at + n], cv[:, at:at + n] = k, v
                o = natten_amd.prefix_attention(q, pk, pv, ck, cv, seq_lens=lens, kernel_size=K)
                h = h + m.proj(o.flatten(-2))
            got.append(h)
            at += n
    assert torch.allclose(torch.cat(got, 1), want, rtol=2e-4, atol=2e-4)


def test_layer_arguments():
    from natten_amd import nn

    plain = nn.NeighborhoodAttention2D(32, 2, 3)
    assert set(plain.state_dict()) == {"qkv.weight", "qkv.bias", "proj.weight", "proj.bias"}
    m = nn.NeighborhoodAttention2D(32, 2, 3, qk_norm=True, rotary=True)
    assert set(m.state_dict()) == set(plain.state_dict()) | {
        f"{a}_norm.{b}" for a in "qk" for b in ("weight", "bias")}
    assert m.rotary_dims == (8, 8) and plain.rotary_dims is None
    assert nn.NeighborhoodAttention3D(64, 2, 3, rotary=(8, 12, 12)).rotary_dims == (8, 12, 12)
    for bad in ((16,), (8, 7), (16, 18), (0, 8), (8.0, 8)):
        with pytest.raises(ValueError, match="rotary must be 2"):
            nn.NeighborhoodAttention2D(32, 2, 3, rotary=bad)
    with pytest.raises(ValueError, match="axes"):
        nn.NeighborhoodAttention3D(8, 2, 3, rotary=True)
    with pytest.raises(ValueError, match="channels"):
        nn.LayerNorm(0)
    assert nn.LayerNorm(4, bias=False).bias is None
    x = torch.randn(1, 4, 4, 32)
    with pytest.raises(RuntimeError, match="HIP"):
        m(x)

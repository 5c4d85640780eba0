"""norm_rotary, cache_append and cache_attention as a model uses them: layers with
``qk_fused`` against those that norm and rotate one after the other and against a
float64 composition, their gradients and graph capture; a text generated one token at
a time from a paged 8-bit cache against the same layers over the whole sequence with
the cache's own rounding; and a generation in one replayed graph."""

import io

import pytest
import torch

from _helpers import DEV, randn
from test_layer_operators import _layer, _reference

F32, BF16 = torch.float32, torch.bfloat16

LAYERS = {
    "1d causal": (1, (2, 40, 32), dict(embed_dim=32, num_heads=2, kernel_size=9, is_causal=True, rotary=True)),
    "2d": (2, (2, 9, 11, 48), dict(embed_dim=48, num_heads=2, kernel_size=5, rotary=(12, 8), rotary_theta=100.0)),
    "2d strided gqa": (2, (1, 12, 10, 64), dict(embed_dim=64, num_heads=4, num_kv_heads=2, kernel_size=3,
                                               stride=2, rotary=True)),
    "3d": (3, (1, 4, 6, 5, 40), dict(embed_dim=40, num_heads=2, kernel_size=3, rotary=True)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(LAYERS))
def test_fused_layers_against_float64(case):
    """float32: as test_layer_operators, every value within 2e-4 of its own or of the
    tensor's largest."""
    rank, shape, kw = LAYERS[case]
    m = _layer(rank, qk_norm=True, qk_fused=True, **kw)
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
def test_fused_layer_beside_the_two_operators():
    """Without qk_fused, with a hook or with unlike eps the layer runs the two operators,
    bit for bit; with it the result differs by the one rounding of q and k that is left
    out, 2^-8 of them, through stages that change values by their own size at most (seven
    stages, as in test_layer_operators)."""
    kw = dict(embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True)
    two, one = (_layer(2, BF16, qk_fused=f, **kw).to(DEV) for f in (False, True))
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    a, b = two(x), one(x)
    assert not torch.equal(a, b)
    assert (a.float() - b.float()).norm() <= 7 * 2 ** -8 * a.float().norm()
    seen = []
    handle = one.q_norm.register_forward_hook(lambda m, i, o: seen.append(o.shape))
    assert torch.equal(one(x), a) and len(seen) == 1
    handle.remove()
    assert torch.equal(one(x), b)
    one.k_norm.eps = two.k_norm.eps = 1e-3
    assert torch.equal(one(x), two(x))


@pytest.mark.gpu
def test_fused_layer_capture():
    m = _layer(2, BF16, embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True, qk_fused=True).to(DEV)
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    g = randn(x.shape, BF16, 2).to(DEV)

    def step():
        out = m(x)
        return [out.detach(), *torch.autograd.grad(out, list(m.parameters()), g)]

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


def _project(m, h, pos, hk):
    import natten_amd

    H, D = m.num_heads, m.head_dim
    if hk == H:
        q, k, v = m._split_qkv(m.qkv(h))
    else:
        q = m.q_proj(h).view(*h.shape[:2], H, D)
        k, v = m.kv_proj(h).view(*h.shape[:2], 2, hk, D).unbind(-3)
    q, k = natten_amd.norm_rotary(q, k, m.q_norm.weight, m.q_norm.bias, m.k_norm.weight, m.k_norm.bias,
                                  positions=pos, axis_dims=m.rotary_dims)
    return q, k, v


def _held(cache, tables, n):
    """Keys and values [B, n, heads, D] that the cache holds, float32."""
    out = []
    for codes, scale in zip(cache[:2], cache[2:]):
        x = codes.view(torch.uint8)[tables.long()].view(codes.dtype).float()
        x = x * scale.view(torch.uint8)[tables.long()].view(scale.dtype).float()[..., None, None]
        out.append(x.transpose(2, 3).flatten(1, 2)[:, :n])
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("hk", [4, 2])
def test_generation_from_a_paged_cache(hk):
    """Texts of unlike lengths through two layers: a padded chunk of prompts, then token
    by token.  What every step attends to is what the cache then holds, so each step's
    output is that of na1d over those keys and values, which differ from the exact ones
    by their rounding alone (half a step of 2^-4, and 2^-10 of the scale's unit)."""
    import natten_amd

    B, T, C, H, K, size = 3, 37, 64, 4, 16, 16
    layers = [_layer(1, embed_dim=C, num_heads=H, num_kv_heads=hk, kernel_size=K, is_causal=True,
                     qk_norm=True, rotary=True, qk_fused=True).to(DEV) for _ in range(2)]
    norms = [natten_amd.nn.LayerNorm(C).to(DEV) for _ in range(2)]
    x = randn((B, T, C), F32, 1).to(DEV)
    caches = [natten_amd.paged_cache(B * 3, hk, C // H, size) for _ in range(2)]
    tables = torch.randperm(B * 3, generator=torch.Generator().manual_seed(1)).view(B, 3).to(DEV)
    have = torch.tensor([12, 5, 9], device=DEV)  # tokens of each prompt, padded in front to 12
    with torch.no_grad():
        at = torch.zeros(B, dtype=torch.long, device=DEV)
        for n, new in ((12, have), *[(1, torch.ones_like(have))] * 20):
            at = at + new
            j = torch.arange(n, device=DEV)
            pos = (at[:, None] - n + j)
            h = x.gather(1, pos.clamp_min(0)[..., None].expand(-1, -1, C))
            for m, nm, cache in zip(layers, norms, caches):
                q, k, v = _project(m, nm(h), pos.clamp_min(0).unsqueeze(-1), hk)
                natten_amd.cache_append(cache, k, v, tables, at, new)
                o = natten_amd.cache_attention(q, cache, tables, at, kernel_size=K)
                for b in range(B):
                    t, real = int(at[b]), int(new[b])
                    keys, vals = (y[b:b + 1, :t].contiguous() for y in _held(cache, tables, t))
                    qs = torch.zeros(1, t, H, C // H, device=DEV)
                    qs[0, t - real:] = q[b, n - real:]
                    want = natten_amd.na1d(qs, keys, vals, kernel_size=min(K, t), is_causal=True)[0, t - real:]
                    assert torch.allclose(o[b, n - real:], want, rtol=1e-5, atol=1e-5)
                    for held, exact in ((keys, k), (vals, v)):
                        e = exact[b, n - real:]
                        off = (held[0, t - real:] - e).abs()
                        assert (off <= e.abs() * 2.0 ** -4 + 2.0 ** -10 * held.abs().max()).all()
                h = h + m.proj(o.flatten(-2))
            assert h.isfinite().all()


@pytest.mark.gpu
def test_generation_in_one_graph():
    """A step with its lengths, positions and cache on the device, replayed token after
    token, against eager steps."""
    import natten_amd

    B, C, H, hk, K, size = 4, 64, 4, 2, 24, 16
    m = _layer(1, BF16, embed_dim=C, num_heads=H, num_kv_heads=hk, kernel_size=K, is_causal=True,
               qk_norm=True, rotary=True, qk_fused=True).to(DEV)
    nm = natten_amd.nn.LayerNorm(C).to(DEV).to(BF16)
    tables = torch.arange(B * 4, device=DEV, dtype=torch.int32).view(B, 4)
    start = torch.tensor([0, 15, 7, 30], dtype=torch.int32, device=DEV)
    state = [dict(h=torch.zeros(B, 1, C, dtype=BF16, device=DEV), lens=start.clone(),
                  cache=natten_amd.paged_cache(B * 4, hk, C // H, size)) for _ in range(2)]

    def step(s):
        s["lens"] += 1
        q, k, v = _project(m, nm(s["h"]), (s["lens"] - 1).view(B, 1, 1), hk)
        natten_amd.cache_append(s["cache"], k, v, tables, s["lens"])
        return s["h"] + m.proj(natten_amd.cache_attention(q, s["cache"], tables, s["lens"], kernel_size=K).flatten(-2))

    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(state[0])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                held = step(state[0])
        torch.cuda.current_stream().wait_stream(side)
        state[0]["lens"].copy_(start)
        for t in state[0]["cache"]:
            t.view(torch.uint8).fill_(127 if t.dtype == torch.float8_e8m0fnu else 0)
        for r in range(20):
            x = randn((B, 1, C), BF16, r).to(DEV)
            for s in state:
                s["h"].copy_(x)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(step(state[1]), held), r
            for a, b in zip(state[0]["cache"], state[1]["cache"]):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), r


def test_fused_layer_arguments():
    from natten_amd import nn

    m = nn.NeighborhoodAttention2D(32, 2, 3, qk_norm=True, rotary=True, qk_fused=True)
    two = nn.NeighborhoodAttention2D(32, 2, 3, qk_norm=True, rotary=True)
    assert m.qk_fused and not two.qk_fused and set(m.state_dict()) == set(two.state_dict())
    for kw in (dict(), dict(qk_norm=True), dict(rotary=True)):
        with pytest.raises(ValueError, match="qk_fused needs"):
            nn.NeighborhoodAttention2D(32, 2, 3, qk_fused=True, **kw)
    with pytest.raises(ValueError, match="up to 256"):
        nn.NeighborhoodAttention1D(512, 1, 3, qk_norm=True, rotary=True, qk_fused=True)
    with pytest.raises(RuntimeError, match="HIP"):
        m(torch.randn(1, 4, 4, 32))
    del two.__dict__["qk_fused"]  # pickled before layers had it
    f = io.BytesIO()
    torch.save(two, f)
    f.seek(0)
    assert torch.load(f, weights_only=False).qk_fused is False


@pytest.mark.gpu
def test_compiled():
    """A compiled step leaves the operators to eager execution: the same bits."""
    import natten_amd

    B, hk, size = 3, 2, 16
    q, k, v = (randn((B, 4, h, 32), BF16, s).to(DEV) for s, h in ((1, 4), (2, hk), (3, hk)))
    w = randn((32,), BF16, 4).to(DEV)
    tables = torch.arange(B * 4, device=DEV).view(B, 4)
    lens = torch.tensor([40, 4, 17], device=DEV)

    def step(cache, q, k, v, lens):
        a, b = natten_amd.norm_rotary(q * 2, k, w, None, w, None, axis_dims=(32,))
        natten_amd.cache_append(cache, b, v, tables, lens)
        return natten_amd.cache_attention(a, cache, tables, lens, kernel_size=20) + 1

    with torch.no_grad():
        caches = [natten_amd.paged_cache(B * 4, hk, 32, size) for _ in range(2)]
        want = step(caches[0], q, k, v, lens)
        assert torch.equal(torch.compile(step, backend="eager")(caches[1], q, k, v, lens), want)
    for a, b in zip(*caches):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.gpu
def test_two_steps_at_once():
    """Two streams, each its own samples and pages of one cache; the same calls one after
    the other."""
    import natten_amd

    B, hk, D, size = 6, 2, 64, 32
    start = randn((2 * B, 300, hk, D), BF16, 1).to(DEV)
    q, k, v = (randn((2 * B, 1, h, D), BF16, s).to(DEV) for s, h in ((2, 8), (3, hk), (4, hk)))
    for width in (11, 64):  # tables of one launch and of two
        tables = torch.randperm(2 * B * 11, generator=torch.Generator().manual_seed(1)).view(2 * B, 11)
        tables = torch.cat([tables, torch.full((2 * B, width - 11), -1)], 1).to(DEV)
        lens = torch.arange(290, 290 + 2 * B, device=DEV)
        outs = []
        for together in (True, False):
            cache = natten_amd.paged_cache(2 * B * 11, hk, D, size)
            natten_amd.cache_append(cache, start, start, tables, lens - 1)
            streams = [torch.cuda.Stream() for _ in "ab"]
            torch.cuda.synchronize()
            got = [None, None]
            for rep in range(5):
                for i, s in enumerate(streams):
                    part = slice(i * B, (i + 1) * B)
                    with torch.cuda.stream(s):
                        natten_amd.cache_append(cache, k[part], v[part], tables[part], lens[part])
                        got[i] = natten_amd.cache_attention(q[part], cache, tables[part], lens[part])
                    if not together:
                        torch.cuda.synchronize()
            torch.cuda.synchronize()
            outs.append((torch.cat(got), *(t.view(torch.uint8) for t in cache)))
        for a, b in zip(*outs):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_more_than_32_bits_of_queries():
    """norm_rotary and its gradients at the end of a tensor of more than 2^31 elements, and
    a prompt's attention into an output of more: the last rows alone, the same bits."""
    import natten_amd

    n, D = (1 << 21) + 77, 128
    w, b = (randn((D,), BF16, s).to(DEV) for s in (1, 2))
    q = torch.empty((1, n, 8, D), dtype=BF16, device=DEV).normal_().requires_grad_(True)
    g = torch.empty_like(q, requires_grad=False).normal_()
    out = natten_amd.norm_rotary(q, None, w, b, axis_dims=(D,))
    dq, = torch.autograd.grad(out, q, g)
    for at in (0, n - 5):
        part = q.detach()[:, at:at + 5].clone().requires_grad_(True)
        pos = torch.arange(at, at + 5, device=DEV).unsqueeze(-1)
        few = natten_amd.norm_rotary(part, None, w, b, positions=pos, axis_dims=(D,))
        assert torch.equal(out[:, at:at + 5], few)
        assert torch.equal(dq[:, at:at + 5], torch.autograd.grad(few, part, g[:, at:at + 5])[0])
    del out, dq, g
    cache = natten_amd.paged_cache(4, 8, D, 16)
    kv = randn((1, 64, 8, D), BF16, 5).to(DEV)
    tables = torch.tensor([[2, 0, 3, 1]], device=DEV)
    with torch.no_grad():
        natten_amd.cache_append(cache, kv, kv, tables, torch.tensor([64], device=DEV))
        # (all but the last 64 of the rows lie before the sequence's start)
        out = natten_amd.cache_attention(q, cache, tables, torch.tensor([64], device=DEV))
        few = natten_amd.cache_attention(q[:, -64:], cache, tables, torch.tensor([64], device=DEV))
    assert torch.allclose(out[:, -64:].float(), few.float(), rtol=2.0 ** -7, atol=2.0 ** -7)
    assert few.abs().max() > 0 and not out[:, :-64].any()


@pytest.mark.gpu
def test_inference_mode():
    """A cache made under inference mode, by both routes, and one made outside it."""
    import natten_amd
    from natten_amd.autograd import fused

    k, q = randn((2, 5, 2, 32), BF16, 1).to(DEV), randn((2, 5, 4, 32), BF16, 2).to(DEV)
    tables, lens = torch.tensor([[0], [1]], device=DEV), torch.tensor([5, 3], device=DEV)

    def step(cache):
        natten_amd.cache_append(cache, k, k, tables, lens)
        return natten_amd.cache_attention(q, cache, tables, lens).clone()

    outside = natten_amd.paged_cache(2, 2, 32, 16)
    outs = [step(outside)]
    with torch.inference_mode():
        outs.append(step(outside))
        outs.append(step(natten_amd.paged_cache(2, 2, 32, 16)))
        with fused.python_autograd():
            outs.append(step(outside))
            outs.append(step(natten_amd.paged_cache(2, 2, 32, 16)))
        inside = natten_amd.paged_cache(2, 2, 32, 16)
        outs.append(torch.compile(step, backend="eager")(inside))
    outs.append(step(inside))
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.gpu
def test_fused_layer_with_unlike_norms():
    """Weights of two types, which one pass does not take, run as without qk_fused."""
    kw = dict(embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True)
    two, one = (_layer(2, BF16, qk_fused=f, **kw).to(DEV) for f in (False, True))
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    for m in (two, one):
        m.q_norm.float()  # (the other's weights stay bfloat16)
    assert torch.equal(one(x), two(x))

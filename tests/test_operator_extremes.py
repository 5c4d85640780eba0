"""Sizes past 32 bits for the layer norm, rotary positions and shared-prefix
attention: tensors and strides whose offsets do not fit 32 bits, against the same
call on a small copy, bit for bit; and the operators under compilation."""

import pytest
import torch

from _helpers import DEV, randn

F32, BF16 = torch.float32, torch.bfloat16


@pytest.mark.gpu
def test_norm_past_32_bits():
    import natten_amd

    rows, c = 540000, 4096  # 2.2e9 elements
    x = torch.empty(rows, c, dtype=BF16, device=DEV)
    g = torch.empty(rows, c, dtype=BF16, device=DEV)
    w, b = (randn((c,), F32, s).to(DEV) for s in (1, 2))
    pick = torch.tensor([0, 7, 262143, 262144, 524287, 524288, rows - 1], device=DEV)
    x.fill_(0.5)
    g.zero_()
    x[pick], g[pick] = randn((7, c), BF16, 3).to(DEV), randn((7, c), BF16, 4).to(DEV)
    x.requires_grad_(True)
    small = x.detach()[pick].requires_grad_(True)
    y, ys = natten_amd.layer_norm(x, w, b), natten_amd.layer_norm(small, w, b)
    assert torch.equal(y[pick], ys)
    (dx,), (ds,) = torch.autograd.grad(y, x, g), torch.autograd.grad(ys, small, g[pick])
    assert torch.equal(dx[pick], ds)
    assert not dx[1].any()
    del y, dx
    # a few rows whose strides pass 32 bits
    view = x.detach().view(-1).as_strided((5, 2, 64), (1 << 29, 1 << 25, 1))
    view.copy_(randn(view.shape, BF16, 5).to(DEV))
    assert torch.equal(natten_amd.layer_norm(view), natten_amd.layer_norm(view.contiguous()))


@pytest.mark.gpu
def test_rotary_past_32_bits():
    import natten_amd

    tokens = 2200000
    q = torch.zeros(1, tokens, 8, 128, dtype=BF16, device=DEV)
    pick = torch.tensor([0, 5, 1048575, 2097151, 2097152, tokens - 1], device=DEV)
    q[0, pick] = randn((6, 8, 128), BF16, 1).to(DEV)
    for dims in ((128,), (46,)):
        out = natten_amd.rotary(q, axis_dims=dims)
        few = natten_amd.rotary(q[:, pick].contiguous(), positions=pick.view(1, -1, 1), axis_dims=dims)
        assert torch.equal(out[:, pick], few)
        assert not out[0, 3].any()
    view = q.view(-1).as_strided((2, 2, 3, 32), (1 << 30, 1 << 29, 1 << 20, 1))
    view.copy_(randn(view.shape, BF16, 2).to(DEV))
    assert torch.equal(natten_amd.rotary(view), natten_amd.rotary(view.contiguous()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_prefix_attention_past_32_bits(dtype):
    """Caches with strides of 2^27 elements and more between their tokens."""
    import natten_amd

    step = 1 << 27
    buf = torch.zeros(41 * step, dtype=dtype, device=DEV)
    B, S, Hk, D = 1, 37, 2, 64
    k = buf.as_strided((B, S, Hk, D), (1, step, 64, 1))
    v = buf.as_strided((B, S, Hk, D), (1, step, 64, 1), 4096)
    pk = buf.as_strided((40, Hk, D), (step, 64, 1), 8192)
    pv = buf.as_strided((40, Hk, D), (step, 64, 1), 16384)
    for t, s in ((k, 1), (v, 2), (pk, 3), (pv, 4)):
        t.copy_(randn(t.shape, dtype, s).to(DEV))
    for L, H in ((1, 4), (3, 40)):  # narrow and wide
        q = randn((B, L, H, D), dtype, 5).to(DEV)
        got = natten_amd.prefix_attention(q, pk, pv, k, v, return_lse=True)
        want = natten_amd.prefix_attention(q, *(t.contiguous() for t in (pk, pv, k, v)), return_lse=True)
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_compiled_calls_run_as_eager():
    import natten_amd

    def f(x, w, pk, pv):
        y = natten_amd.layer_norm(x, w, eps=1e-6).view(2, 9, 4, 16)
        q, k = natten_amd.rotary(y, y)
        return q + k

    def serve(q, pk, pv):
        with torch.no_grad():
            return natten_amd.prefix_attention(q * 2, pk, pv) + 1

    x, w = randn((2, 9, 64), F32, 1).to(DEV).requires_grad_(True), randn((64,), F32, 2).to(DEV)
    pk, pv = (randn((5, 2, 16), F32, s).to(DEV) for s in (3, 4))
    want, got = f(x, w, pk, pv), torch.compile(f)(x, w, pk, pv)
    assert torch.equal(got, want)
    g = randn(want.shape, F32, 5).to(DEV)
    assert torch.equal(torch.autograd.grad(got, x, g)[0], torch.autograd.grad(want, x, g)[0])
    q = want.detach()
    assert torch.equal(torch.compile(serve)(q, pk, pv), serve(q, pk, pv))


def test_launches_end_at_their_limits():
    """What does not fit one launch is refused before anything is launched."""
    from natten_amd._core import _lib

    lib = _lib.load()
    somewhere = 256  # an address that a refused call does not touch

    def rotary(**kw):
        p = _lib.NaRotaryParams(**{**dict(batch=1, heads=1, kv_heads=0, head_dim=1024, dtype=0,
                                          n_axes=1, theta=1e4), **kw})
        p.extent[0], p.extent[1], p.extent[2], p.axis_dim[0] = 1, 1, 5, 16
        return lib.na_rotary(p, *([somewhere] * 5), None)

    if not torch.cuda.is_available():  # here nothing could be launched
        assert rotary(heads=1 << 19) == 2 and b"one launch" in lib.na_last_error()
        assert rotary(batch=1 << 27, heads=64) == 2 and b"one launch" in lib.na_last_error()

    def prefix(**kw):
        p = _lib.NaPrefixParams(**{**dict(batch=1, tokens=1, heads=16, kv_heads=16, head_dim=16,
                                          dtype=2, prefix=5, capacity=7, scale=0.25), **kw})
        return lib.na_prefix_fwd(p, *([None] * 8), 0, None)

    assert prefix(batch=1 << 25) == 2 and b"one launch" in lib.na_last_error()
    assert prefix(batch=1 << 25, kv_heads=1, head_dim=256) == 2


def test_a_long_prompt_takes_a_workspace_of_few_slots():
    """Rows that fill the chip many times over meet their own keys in few chunks: the
    workspace is a small number of float32 rows per query, whatever the length."""
    from natten_amd._core import _lib

    lib = _lib.load()

    def slots(tokens, capacity, batch=1):
        p = _lib.NaPrefixParams(batch=batch, tokens=tokens, heads=32, kv_heads=8, head_dim=128,
                                dtype=2, prefix=64, capacity=capacity, scale=0.1)
        return lib.na_prefix_workspace_bytes(p) / (batch * tokens * 32 * (128 + 2) * 4)

    assert slots(8192, 131072) < 10
    assert slots(2048, 32768) < 20
    assert slots(1, 32768) > 20  # few rows: the keys are shared out

"""norm_rotary without tokens or without heads: gradients are zeros, and no call ends the
process."""

import os
import subprocess
import sys

import pytest
import torch

from _helpers import DEV

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "natten-mlx_amd")

SIZES = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from natten_amd._core import _lib
r = _lib.NaRotaryParams(batch=int(sys.argv[5]), heads=4, kv_heads=1, head_dim=16, dtype=2, n_axes=1, theta=1e4)
r.extent[:] = [int(x) for x in sys.argv[2:5]]
r.axis_dim[0] = 16
p = _lib.NaNormRotaryParams(rotary=r, weight_dtype=0, eps=1e-5)
print(_lib.load().na_norm_rotary_bwd_workspace_bytes(p))
"""


@pytest.mark.parametrize("extent, batch", [((1, 1, 0), 2), ((1, 0, 3), 2), ((0, 1, 5), 2), ((0, 0, 0), 2),
                                           ((1, 1 << 16, 1 << 16), 0), ((1, 0, 0), 0)], ids=str)
def test_sizes_of_an_empty_grid(extent, batch):
    """In a process of its own, which a division by an extent of zero would end."""
    run = subprocess.run([sys.executable, "-c", SIZES, PKG, *map(str, extent), str(batch)],
                         capture_output=True, text=True)
    assert run.returncode == 0, (run.returncode, run.stderr)
    assert run.stdout.split()[-1] == "0"


@pytest.mark.gpu
@pytest.mark.parametrize("lead", [(2, 0), (2, 3, 0), (2, 0, 3), (0, 5), (1, 2, 0, 4), (0, 0),
                                  (0, 1 << 16, 1 << 16)], ids=str)
@pytest.mark.parametrize("twin", [False, True])
def test_gradients_without_tokens(lead, twin):
    import natten_amd
    import natten_amd.autograd.fused as AF

    q, k = (torch.empty((*lead, h, 16), device=DEV, requires_grad=True) for h in (4, 1))
    w = [torch.ones(16, device=DEV, requires_grad=True) for _ in range(4)]
    with AF.python_autograd(twin):
        out = natten_amd.norm_rotary(q, k, *w)
        assert out[0].shape == q.shape and out[1].shape == k.shape
        grads = torch.autograd.grad(out[0].sum() + out[1].sum(), (q, k, *w), retain_graph=True)
        alone, = torch.autograd.grad(out[0].sum(), q)
    assert grads[0].shape == q.shape and grads[1].shape == k.shape and alone.shape == q.shape
    for g in grads[2:]:
        assert g.shape == (16,) and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("twin", [False, True])
@pytest.mark.parametrize("key", [False, True])
def test_gradients_without_heads(key, twin, dtype):
    """Not what the memory held before: blocks of NaN of every size are there to be taken."""
    import natten_amd
    import natten_amd.autograd.fused as AF

    q = torch.empty((2, 3, 0, 16), device=DEV, dtype=dtype, requires_grad=True)
    k = q.detach().clone().requires_grad_(True) if key else None
    w = [torch.ones(16, device=DEV, dtype=dtype, requires_grad=True) for _ in range(4 if key else 2)]
    dirty = [torch.full((16,), float("nan"), device=DEV, dtype=dtype) for _ in range(64)]
    torch.cuda.synchronize()
    del dirty
    with AF.python_autograd(twin):
        out = natten_amd.norm_rotary(q, k, *w)
        grads = torch.autograd.grad(sum(o.sum() for o in (out if key else (out,))), w)
    for g in grads:
        assert g.shape == (16,) and g.isfinite().all() and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv_heads", [(0, 3), (3, 0)])
@pytest.mark.parametrize("twin", [False, True])
def test_heads_of_one_tensor_alone(heads, kv_heads, twin):
    """The other's weights get zeros, and what has heads what it gets by itself."""
    import natten_amd
    import natten_amd.autograd.fused as AF
    from _helpers import randn

    q, k = (randn((2, 5, h, 16), seed=s).to(DEV).requires_grad_(True) for s, h in ((1, heads), (2, kv_heads)))
    w = [randn((16,), seed=3 + i).to(DEV).requires_grad_(True) for i in range(4)]
    some, ws, none = (q, w[:2], w[2:]) if heads else (k, w[2:], w[:2])
    with AF.python_autograd(twin):
        out = natten_amd.norm_rotary(q, k, *w)
        part = out[0] if heads else out[1]
        g = torch.autograd.grad(out[0].square().sum() + out[1].square().sum(), (some, *ws, *none))
        alone = natten_amd.norm_rotary(some, q_weight=ws[0], q_bias=ws[1])
        want = torch.autograd.grad(alone.square().sum(), (some, *ws))
    assert torch.equal(part, alone)
    for a, b in zip(g, want):
        assert torch.equal(a, b)
    assert not g[3].any() and not g[4].any()

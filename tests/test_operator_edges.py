"""Calls at the edges of what the layer norm, rotary positions and shared-prefix
attention document: the widest windows of the C ABI."""

import pytest
import torch

from _helpers import DEV
from test_prefix import _make, _near, _reference

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


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

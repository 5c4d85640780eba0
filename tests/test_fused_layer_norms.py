"""Layers with ``qk_fused`` whose norms are not the layer's plain ones: they are called
themselves, as without it."""

import pytest
import torch

from _helpers import DEV, randn
from test_layer_operators import _layer

BF16 = torch.bfloat16
KW = dict(embed_dim=64, num_heads=2, kernel_size=7, qk_norm=True, rotary=True)


class Doubled(torch.nn.Module):
    def forward(self, x):
        return 2 * x


def _without(m, name):
    setattr(m, name, None)
    return m


def _own_forward(m):
    m.forward = lambda x: 3 * x
    return m


NORMS = {
    "identity": lambda m: torch.nn.Identity(),
    "another module": lambda m: Doubled(),
    "torch's, plain": lambda m: torch.nn.LayerNorm(32),
    "torch's, no weight": lambda m: torch.nn.LayerNorm(32, elementwise_affine=False),
    "a forward of its own": _own_forward,
    "a subclass": lambda m: type("Mine", (type(m),), {})(32),
}


@pytest.mark.parametrize("which", ["q_norm", "k_norm", "both"])
@pytest.mark.parametrize("norm", list(NORMS))
def test_replaced_norms_are_not_fused(norm, which):
    m = _layer(2, qk_fused=True, **KW)
    assert m._fuses_norms()
    for n in ("q_norm", "k_norm"):
        if which in (n, "both"):
            setattr(m, n, NORMS[norm](getattr(m, n)))
    assert not m._fuses_norms()
    with pytest.raises(RuntimeError, match="HIP"):  # (the first kernel, whichever it is)
        m(torch.randn(1, 8, 8, 64))


@pytest.mark.parametrize("names", [("weight",), ("bias",), ("weight", "bias")])
def test_norms_without_weights_or_biases(names):
    m = _layer(2, qk_fused=True, **KW)
    for n in names:
        _without(m.q_norm, n)
    assert m._fuses_norms()
    m.k_norm.half()
    assert m._fuses_norms() == (len(names) == 2)  # (one type is left)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", list(NORMS))
def test_replaced_norms_run(norm):
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    outs = []
    for fused in (False, True):
        m = _layer(2, BF16, qk_fused=fused, **KW)
        m.k_norm = NORMS[norm](m.k_norm)
        outs.append(m.to(DEV, BF16)(x))
    assert torch.equal(*outs)


@pytest.mark.gpu
@pytest.mark.parametrize("names", [("weight",), ("bias",), ("weight", "bias")])
def test_norms_without_weights_run(names):
    """The one rounding that the fused pass leaves out, as in test_serving_operators."""
    x = randn((2, 16, 14, 64), BF16, 1).to(DEV)
    outs = []
    for fused in (False, True):
        m = _layer(2, BF16, qk_fused=fused, **KW).to(DEV)
        for n in names:
            _without(m.q_norm, n)
        outs.append(m(x).float())
    assert (outs[0] - outs[1]).norm() <= 7 * 2 ** -8 * outs[0].norm()

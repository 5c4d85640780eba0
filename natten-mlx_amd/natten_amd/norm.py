"""Layer norm over the last dimension, for a layer's input and for its queries
and keys (no counterpart in the reference, whose models take their framework's).

With the built-in library it is an operator with its autograd node in C++
(``csrc/na_torch.cpp``); ``_Norm`` below is the same op as a Python Function
over the same kernels, for compiled and transformed code and under
``python_autograd()``.
"""

from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from ._core import _lib
from ._core import hip
from .autograd import fused as _fused


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, eps):
        y, stats = hip.norm_forward(x, w, b, eps)
        ctx.save_for_backward(x, w, b, stats)
        ctx.eps = eps
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, w, b, stats = ctx.saved_tensors
        return (*hip.norm_backward(x, w, b, dy, stats, ctx.eps, ctx.needs_input_grad), None)


def layer_norm(input: torch.Tensor, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """``(input - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    input ``[..., C]`` in float32, float16 or bfloat16, C from 1 to 16384; its rows
    may be a view, such as one part of a packed projection ``[..., 3, H, D]``, which
    is read in place.  weight and bias ``[C]``, either or both left out, in input's
    type or float32 (both in the same).  Mean, variance and the gradients' sums are
    float32; the output has input's type.  Differentiable once in each of the three;
    the weight's gradient is summed in a fixed order.
    """
    if input.ndim < 1 or not 1 <= input.shape[-1] <= _lib.NORM_MAX_CHANNELS:
        raise ValueError(f"layer_norm expects [..., C] with C from 1 to {_lib.NORM_MAX_CHANNELS}, "
                         f"got shape {tuple(input.shape)}.")
    wdt = None
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.ndim != 1 or t.shape[0] != input.shape[-1]:
            raise ValueError(f"{name} must have shape [{input.shape[-1]}], got {tuple(t.shape)}.")
        if t.dtype != input.dtype and t.dtype != torch.float32:
            raise ValueError(f"{name} must be {input.dtype} or float32, got {t.dtype}.")
        if wdt is not None and t.dtype != wdt:
            raise ValueError(f"weight and bias must have the same dtype, got {wdt} and {t.dtype}.")
        wdt = t.dtype
    if not eps >= 0.0:
        raise ValueError(f"eps must be >= 0, got {eps}.")
    if not _fused._py_autograd:
        op = _lib.node_op("norm", input, input if weight is None else weight)
        if op is not None:
            return op(input, weight, bias, eps, _lib.stream_of(input))
    return _Norm.apply(input, weight, bias, eps)


__all__ = ["layer_norm"]

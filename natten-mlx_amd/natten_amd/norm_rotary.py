"""The layer norm of queries and keys with their rotary positions in one pass, for
layers that norm each head before they turn it (no counterpart in the reference).

With the built-in library it is an operator with its autograd node in C++
(``csrc/na_torch.cpp``); ``_NormRotary`` below is the same op as a Python Function
over the same kernels, for compiled and transformed code and under
``python_autograd()``.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch
from torch.autograd.function import once_differentiable

from ._core import _lib
from ._core import hip
from .autograd import fused as _fused
from .rotary import _check as _check_rotary


class _NormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, wq, bq, wk, bk, positions, args, eps):
        ctx.save_for_backward(q, k, wq, bq, wk, bk, positions)
        ctx.args, ctx.eps = args, eps
        ctx.set_materialize_grads(False)
        return hip.norm_rotary_forward(q, k, wq, bq, wk, bk, positions, args, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        return (*hip.norm_rotary_backward(*ctx.saved_tensors, ctx.args, ctx.eps, gq, gk,
                                          ctx.needs_input_grad[:6]), None, None, None)


def _check(query, key, weights, eps):
    d = query.shape[-1]
    if d > _lib.NORM_ROTARY_MAX_HEAD_DIM:
        raise ValueError(f"norm_rotary takes up to {_lib.NORM_ROTARY_MAX_HEAD_DIM} channels, got {d}; "
                         "wider heads take layer_norm and rotary.")
    wdt = None
    for name, t in weights:
        if t is None:
            continue
        if t.ndim != 1 or t.shape[0] != d:
            raise ValueError(f"{name} must have shape [{d}], got {tuple(t.shape)}.")
        if t.dtype != query.dtype and t.dtype != torch.float32:
            raise ValueError(f"{name} must be {query.dtype} or float32, got {t.dtype}.")
        if wdt is not None and t.dtype != wdt:
            raise ValueError(f"weights and biases must have the same dtype, got {wdt} and {t.dtype}.")
        if key is None and name[0] == "k":
            raise ValueError(f"{name} belongs to key, which is missing.")
        wdt = t.dtype
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be >= 0 and finite, got {eps}.")


def norm_rotary(query: torch.Tensor, key: Optional[torch.Tensor] = None,
                q_weight: Optional[torch.Tensor] = None, q_bias: Optional[torch.Tensor] = None,
                k_weight: Optional[torch.Tensor] = None, k_bias: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None,
                axis_dims: Optional[Sequence[int]] = None, theta: float = 10000.0,
                interleaved: bool = False, eps: float = 1e-5
                ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``rotary(layer_norm(query, q_weight, q_bias, eps), layer_norm(key, k_weight,
    k_bias, eps), positions, axis_dims, theta, interleaved)`` in one pass: every head
    of queries ``[B, *spatial, H, D]`` (and keys ``[B, *spatial, H_kv, D]``) is normed over
    its D channels, then turned by its token's position.  With a key, ``(query, key)``.

    D up to 256; positions, ``axis_dims``, ``theta`` and ``interleaved`` as ``rotary``
    takes them.  Weights and biases ``[D]``, each of them left out or all of one type,
    query's or float32; the heads of a tensor share them.  Inputs may be views, such as
    parts of a packed projection; results are contiguous, in query's type, and rounded
    once (the two operators after each other round twice).  Differentiable once in
    queries, keys, weights and biases; the weights' gradients are summed in a fixed
    order.
    """
    dims = _check_rotary(query, key, positions, axis_dims, theta)
    _check(query, key, (("q_weight", q_weight), ("q_bias", q_bias), ("k_weight", k_weight),
                        ("k_bias", k_bias)), eps)
    if positions is not None and positions.ndim == query.ndim - 1 and positions.shape[0] == 1:
        positions = positions[0]
    if not _fused._py_autograd:
        op = _lib.node_op("norm_rotary", query, query if key is None else key)
        if op is not None:
            q, k = op(query, key, q_weight, q_bias, k_weight, k_bias, positions, dims, theta,
                      interleaved, eps, _lib.stream_of(query))
            return q if key is None else (q, k)
    q, k = _NormRotary.apply(query, key, q_weight, q_bias, k_weight, k_bias, positions,
                             (dims, theta, interleaved), eps)
    return q if key is None else (q, k)


__all__ = ["norm_rotary"]

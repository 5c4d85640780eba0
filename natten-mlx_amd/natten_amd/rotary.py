"""Rotary positions by axis (time, height, width) of queries and keys, for
neighborhood attention over sequences, images and videos (no counterpart in the
reference).

With the built-in library it is an operator with its autograd node in C++
(``csrc/na_torch.cpp``); ``_Rotary`` below is the same op as a Python Function
over the same kernel, for compiled and transformed code and under
``python_autograd()``.
"""

from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from ._core import _lib
from ._core import hip
from .autograd import fused as _fused


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, args, inverse):
        ctx.save_for_backward(positions)
        ctx.args, ctx.inverse = args, inverse
        ctx.set_materialize_grads(False)
        return hip.rotary(q, k, positions, *args, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        gq, gk = (g if need else None for g, need in zip((gq, gk), ctx.needs_input_grad))
        if gq is None and gk is None:
            return None, None, None, None, None
        (positions,) = ctx.saved_tensors
        return (*_Rotary.apply(gq, gk, positions, ctx.args, not ctx.inverse), None, None, None)


def rotary_axis_dims(head_dim: int, n_axes: int) -> Tuple[int, ...]:
    """``head_dim`` channels shared out evenly over ``n_axes`` axes in pairs, the
    last axes taking a pair more where they do not divide: 64 over three axes is
    (20, 22, 22)."""
    if n_axes < 1 or head_dim % 2 or head_dim < 2 * n_axes:
        raise ValueError(f"head_dim ({head_dim}) must be even and hold a pair for each of "
                         f"{n_axes} axes; pass axis_dims to rotate a part of it.")
    pairs = head_dim // 2
    return tuple(2 * (pairs * (a + 1) // n_axes - pairs * a // n_axes) for a in range(n_axes))


def _check(query, key, positions, axis_dims, theta):
    shape = query.shape
    if len(shape) not in (4, 5, 6):
        raise ValueError("rotary expects [B, *spatial, heads, dim] with one to three spatial "
                         f"axes, got shape {tuple(shape)}.")
    d = shape[-1]
    if d > _lib.MAX_HEAD_DIM:
        raise ValueError(f"rotary takes up to {_lib.MAX_HEAD_DIM} channels, got {d}.")
    lead = shape[:-2]
    if key is not None:
        ks = key.shape
        if len(ks) != len(shape) or ks[:-2] != lead:
            raise ValueError(f"key must have query's batch and spatial shape {tuple(lead)}, got "
                             f"{tuple(ks)}.")
        if ks[-1] != d:
            raise ValueError(f"Head dim must match: Q has {d}, K has {ks[-1]}.")
        if key.dtype != query.dtype:
            raise ValueError(f"query and key must have the same dtype, got {query.dtype} and "
                             f"{key.dtype}.")
    n = len(lead) - 1
    if positions is not None:
        *at, n = positions.shape or (0,)
        at = tuple(at)
        if at != lead and at != lead[1:] and at != (1, *lead[1:]):
            raise ValueError(f"positions must be [*spatial, axes] or [B, *spatial, axes] for "
                             f"tokens {tuple(lead)}, got {tuple(positions.shape)}.")
        if not 1 <= n <= _lib.ROTARY_MAX_AXES:
            raise ValueError(f"positions must have 1 to {_lib.ROTARY_MAX_AXES} axes, got {n}.")
        if positions.dtype not in _lib.POSITIONS:
            raise ValueError("positions must be int32, int64, float32 or float64, got "
                             f"{positions.dtype}.")
        if positions.requires_grad:
            raise ValueError("positions are not differentiable; pass them detached.")
    dims = rotary_axis_dims(d, n) if axis_dims is None else tuple(axis_dims)
    if len(dims) != n:
        raise ValueError(f"axis_dims must have one entry per axis ({n}), got {dims}.")
    total = 0
    for a in dims:
        if not isinstance(a, int) or a < 2 or a % 2:
            raise ValueError(f"axis_dims must be positive even ints, got {dims}.")
        total += a
    if total > min(d, _lib.ROTARY_MAX_CHANNELS):
        raise ValueError(f"axis_dims {dims} rotate {total} channels of {d} "
                         f"(at most {_lib.ROTARY_MAX_CHANNELS}).")
    if not (theta > 0.0 and math.isfinite(theta)):
        raise ValueError(f"theta must be positive and finite, got {theta}.")
    return dims


def rotary(query: torch.Tensor, key: Optional[torch.Tensor] = None,
           positions: Optional[torch.Tensor] = None,
           axis_dims: Optional[Sequence[int]] = None, theta: float = 10000.0,
           interleaved: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Queries ``[B, *spatial, H, D]`` (and keys ``[B, *spatial, H_kv, D]``) rotated
    by their tokens' positions, in one launch; with a key, ``(query, key)``.

    Axis a owns ``axis_dims[a]`` channels, the axes one after the other (default:
    all channels, shared out by ``rotary_axis_dims``); channels behind the last
    axis pass through.  Its pair i turns by ``position * theta ** (-2 i /
    axis_dims[a])``; pairs lie half an axis apart, or side by side with
    ``interleaved``.  A token's positions are its coordinates on the spatial grid,
    or ``positions[..., a]``: ``[*spatial, axes]``, or ``[B, *spatial, axes]``
    (int32, int64, float32 or float64; one to four axes), as for tokens generated
    one at a time or for images inside a text.  Angles are formed in float64.
    Inputs may be views, such as parts of a packed projection; results are
    contiguous.  Differentiable in query and key, any number of times.
    """
    dims = _check(query, key, positions, axis_dims, theta)
    if positions is not None and positions.ndim == query.ndim - 1 and positions.shape[0] == 1:
        positions = positions[0]
    if not _fused._py_autograd:
        op = _lib.node_op("rotary", query, query if key is None else key)
        if op is not None:
            q, k = op(query, key, positions, dims, theta, interleaved, False,
                      _lib.stream_of(query))
            return q if key is None else (q, k)
    q, k = _Rotary.apply(query, key, positions, (dims, theta, interleaved), False)
    return q if key is None else (q, k)


__all__ = ["rotary", "rotary_axis_dims"]

"""Serving: attention of a batch's newest tokens against key/value caches whose
prefix the whole batch shares (no counterpart in the reference).

It is causal 1D neighborhood attention at the end of a sequence, joined to tokens
that every query sees -- ``na1d(..., is_causal=True, additional_keys=...)`` at its
last rows -- with the caches as they lie and one copy of the shared tokens, whose
keys are read once for all samples (``csrc/na_prefix.hip``).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from ._core import _lib
from ._core import hip
from .autograd import fused as _fused


def _check(query, pk, pv, key, value, seq_lens, kernel_size, scale):
    shape, dtype = query.shape, query.dtype
    if len(shape) != 4:
        raise ValueError(f"query must be [B, L, heads, dim], got {tuple(shape)}.")
    b, _, h, d = shape
    ps = pk.shape
    if len(ps) != 3 or ps != pv.shape or ps[2] != d or ps[1] < 1:
        raise ValueError(f"prefix_key and prefix_value must be [N, heads_kv, {d}], got "
                         f"{tuple(ps)} and {tuple(pv.shape)}.")
    hk = ps[1]
    if h < 1 or h % hk:
        raise ValueError(f"heads_q ({h}) must be divisible by heads_kv ({hk}) for GQA.")
    if d < 8 or d % 8 or d > _lib.PREFIX_MAX_HEAD_DIM:
        raise ValueError(f"head dim must be a multiple of 8 up to {_lib.PREFIX_MAX_HEAD_DIM}, got {d}.")
    if (key is None) != (value is None):
        raise ValueError("key and value must both be provided or both None.")
    tensors = (pk, pv)
    if key is not None:
        tensors = (pk, pv, key, value)
        ks = key.shape
        if len(ks) != 4 or ks != value.shape or ks[0] != b or ks[2] != hk or ks[3] != d:
            raise ValueError(f"key and value must be [{b}, S, {hk}, {d}], got {tuple(ks)} and "
                             f"{tuple(value.shape)}.")
    for t in tensors:
        if t.dtype != dtype:
            raise ValueError(f"keys and values must have query's dtype {dtype}, got {t.dtype}.")
    if seq_lens is not None:
        if key is None:
            raise ValueError("seq_lens are the lengths of key and value, which are missing.")
        if seq_lens.ndim != 1 or seq_lens.shape[0] != b:
            raise ValueError(f"seq_lens must be a 1-D array of length B={b}, got shape "
                             f"{tuple(seq_lens.shape)}.")
        if seq_lens.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"seq_lens must be int32 or int64, got {seq_lens.dtype}.")
    if kernel_size is not None and (not isinstance(kernel_size, int) or kernel_size < 1):
        raise ValueError(f"kernel_size must be a positive int or None, got {kernel_size!r}.")
    if scale is not None and not (scale > 0.0 and math.isfinite(scale)):
        raise ValueError(f"scale must be positive and finite, got {scale}.")


class _Prefix(torch.autograd.Function):
    """The call outside the operator: a Function without derivatives, so that
    forward-mode levels and torch.func transforms are refused, not passed by."""

    @staticmethod
    def forward(ctx, q, pk, pv, k, v, lens, window, scale, want_lse):
        return hip.prefix_forward(q, pk, pv, k, v, lens, window, scale, want_lse)


def _host_lens(seq_lens, capacity, device):
    # lengths change with every generated token: nothing is kept of them
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("seq_lens on the host cannot be captured in a graph: pass them on "
                               "query's device")
    host = seq_lens.tolist()
    if host and (min(host) < 0 or max(host) > capacity):
        raise ValueError(f"All seq_lens must be in [0, {capacity}], got {min(host)} to {max(host)}.")
    return seq_lens.to(torch.int32).to(device)


def prefix_attention(query: torch.Tensor, prefix_key: torch.Tensor, prefix_value: torch.Tensor,
                     key: Optional[torch.Tensor] = None, value: Optional[torch.Tensor] = None,
                     seq_lens: Optional[torch.Tensor] = None, kernel_size: Optional[int] = None,
                     scale: Optional[float] = None, return_lse: bool = False
                     ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The batch's newest tokens ``[B, L, H, D]`` (L = 1: one generated token each)
    attend to shared tokens ``[N, H_kv, D]`` and to their samples' own caches
    ``[B, S, H_kv, D]``.

    ``seq_lens[b]`` (default S) counts the valid own tokens, the new ones among
    them: query j of sample b is own token ``t = seq_lens[b] - L + j``.  It sees every
    prefix token and the own tokens up to t; with ``kernel_size`` the last
    ``kernel_size`` of them only, the causal window of ``na1d``; a query before the
    sequence's start (t < 0) sees the prefix alone.  What a cache holds behind
    ``seq_lens[b]`` is not read.  Lengths on the device are taken as they are,
    clamped to ``[0, S]`` there (no synchronisation); lengths on the host are checked
    and copied at every call, which waits for the stream; under graph capture they are
    refused.

    float32, float16 or bfloat16, all tensors alike; D a multiple of 8 up to 256;
    query heads share key/value heads as in ``na1d``.  Caches and queries may be
    views of any strides whose channels are adjacent, such as heads-first caches.
    The output has query's type; the LSE (``return_lse``) is float32 ``[B, L, H]``,
    ready for ``merge_attentions``.  A query that sees no key gets zeros and -inf.

    There is no derivative: inputs that require grad are refused outside
    ``torch.no_grad()``, tangents of forward mode and torch.func transforms always.
    To train with shared tokens, pass them to ``na1d`` as
    ``additional_keys`` expanded over the batch.
    """
    _check(query, prefix_key, prefix_value, key, value, seq_lens, kernel_size, scale)
    scale = query.shape[-1] ** -0.5 if scale is None else float(scale)
    if seq_lens is not None and not seq_lens.is_cuda and query.is_cuda:
        seq_lens = _host_lens(seq_lens, key.shape[1], query.device)
    window = 0 if kernel_size is None else kernel_size
    op = None if _fused._py_autograd else _lib.node_op("prefix", query, prefix_key)
    if op is not None:
        out, lse = op(query, prefix_key, prefix_value, key, value, seq_lens, window, scale,
                      return_lse, _lib.stream_of(query))
    else:
        if torch.is_grad_enabled() and any(
                t is not None and t.requires_grad
                for t in (query, prefix_key, prefix_value, key, value)):
            raise RuntimeError("prefix_attention serves: it has no backward (under torch.no_grad(), "
                               "or train with the prefix as additional_keys of na1d)")
        if seq_lens is not None:
            seq_lens = seq_lens.clamp(0, key.shape[1]).to(torch.int32)
        out, lse = _Prefix.apply(query, prefix_key, prefix_value, key, value, seq_lens, window, scale,
                                 return_lse)
    return (out, lse) if return_lse else out


__all__ = ["prefix_attention"]

"""Serving: keys and values in pages of 8-bit elements, tokens appended to them and
attention over them (no counterpart in the reference).

``cache_attention`` is causal 1D neighborhood attention at the end of a sequence --
``na1d(..., is_causal=True)`` at its last rows -- whose keys and values lie in a paged
cache at half the bytes of 16-bit ones (``csrc/na_cache.hip``,
``csrc/na_cache_attend.hip``).
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from ._core import _lib
from ._core import hip
from .autograd import fused as _fused
from .prefix import _host_lens


class PagedCache(NamedTuple):
    """Keys and values ``[pages, H_kv, page_size, D]`` in float8_e4m3fn and the scales of
    each page and head ``[pages, H_kv]`` in float8_e8m0fnu (a power of two): an element
    stands for its value times its page's and head's scale.  Scales lie in ``[2^-117,
    2^119]``, as ``cache_append`` writes them; smaller ones are taken as 2^-117, larger
    ones and NaN as 2^119.

    Which page holds which tokens is the caller's: a table ``[B, M]`` says that token i
    of sample b lies in slot ``i % page_size`` of page ``tables[b, i // page_size]``.
    Samples may share pages that are only read; a page to be appended to belongs to one
    sample (copy it first: ``for t in cache: t[new] = t[old]``, on ``t.view(torch.uint8)``
    for tensors of indices).
    """

    key: torch.Tensor
    value: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor


def paged_cache(pages: int, heads: int, dim: int, page_size: int = 64,
                device: Union[str, torch.device] = "cuda") -> PagedCache:
    """An empty ``PagedCache``: ``heads`` key/value heads of ``dim`` channels, a multiple
    of 16 up to 256; ``page_size`` 16, 32, 64 or 128 tokens."""
    for name, n, low in (("pages", pages, 0), ("heads", heads, 1)):
        if not isinstance(n, int) or n < low:
            raise ValueError(f"{name} must be an int of at least {low}, got {n!r}.")
    _check_sizes(dim, page_size)
    codes = [torch.zeros((pages, heads, page_size, dim), dtype=torch.uint8, device=device)
             .view(torch.float8_e4m3fn) for _ in "kv"]
    scales = [torch.full((pages, heads), 127, dtype=torch.uint8, device=device)
              .view(torch.float8_e8m0fnu) for _ in "kv"]
    return PagedCache(*codes, *scales)


def _check_sizes(dim, page_size):
    if not isinstance(dim, int) or dim < 16 or dim % 16 or dim > _lib.CACHE_MAX_HEAD_DIM:
        raise ValueError(f"head dim must be a multiple of 16 up to {_lib.CACHE_MAX_HEAD_DIM}, "
                         f"got {dim}.")
    if page_size not in _lib.CACHE_PAGE_SIZES:
        raise ValueError(f"page_size must be one of {_lib.CACHE_PAGE_SIZES}, got {page_size}.")


_DTYPES = (torch.float8_e4m3fn,) * 2 + (torch.float8_e8m0fnu,) * 2


def _check_cache(cache):
    """The shape ``(pages, heads, page_size, dim)``."""
    if not isinstance(cache, tuple) or len(cache) != 4:
        raise ValueError(f"cache must be a PagedCache, got {type(cache).__name__}.")
    k, v, ks, vs = cache
    shape = tuple(k.shape)
    if len(shape) != 4 or v.shape != shape or shape[1] < 1:
        raise ValueError(f"cache.key and cache.value must be [pages, heads, page_size, dim], got "
                         f"{shape} and {tuple(v.shape)}.")
    pages = shape[:2]
    if ks.shape != pages or vs.shape != pages:
        raise ValueError(f"cache.key_scale and cache.value_scale must be {pages}, got "
                         f"{tuple(ks.shape)} and {tuple(vs.shape)}.")
    if (k.dtype, v.dtype, ks.dtype, vs.dtype) != _DTYPES:
        raise ValueError("cache must hold float8_e4m3fn and float8_e8m0fnu, got "
                         f"{[str(t.dtype) for t in cache]}.")
    _check_sizes(shape[3], shape[2])
    flat = shape[1] * shape[2] * shape[3] < 1 << 31
    for t in (k, v):  # (a copy would not be the cache)
        if flat and t.is_contiguous() and not t.data_ptr() % 16 or not shape[0]:
            continue
        st = [s if n > 1 else 0 for n, s in zip(shape, t.stride())]
        if t.data_ptr() % 16 or st[3] != 1 or any(s % 16 for s in st[:3]):
            raise ValueError("cache.key and cache.value must have adjacent channels and rows that "
                             f"start at multiples of 16, got strides {t.stride()}.")
        if st[0] >= 1 << 31 or st[2] >= 1 << 24:
            raise ValueError("cache.key and cache.value must have strides below 2^31 from page to "
                             f"page and 2^24 from token to token, got {t.stride()}.")
    return shape


def _check_lens(name, t, b):
    if t.ndim != 1 or t.shape[0] != b:
        raise ValueError(f"{name} must be a 1-D array of length B={b}, got shape {tuple(t.shape)}.")
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64, got {t.dtype}.")


def _check_tables(tables, b, page_size):
    if tables.ndim != 2 or tables.shape[0] != b:
        raise ValueError(f"tables must be [{b}, pages of a sample], got {tuple(tables.shape)}.")
    if tables.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tables must be int32 or int64, got {tables.dtype}.")
    if tables.shape[1] * page_size > 1 << 30:
        raise ValueError(f"a sample holds up to 2^30 tokens, got {tables.shape[1]} pages of {page_size}.")


def _narrow(t, low, high):
    """Integers on the device as int32; 64-bit ones are clamped before they are narrowed."""
    return t.clamp(low, high).to(torch.int32) if t.dtype == torch.int64 else t


def _no_derivative(what, tensors):
    """Refuses inputs whose derivatives the caller asks for."""
    for t in tensors:
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f"{what} serves: it has no backward (under torch.no_grad(), or train "
                               "with na1d)")
    if torch._C._functorch.maybe_current_level() is not None:
        raise RuntimeError(f"{what} cannot be transformed by functorch (torch.func)")
    if torch.autograd.forward_ad._current_level >= 0 and any(
            torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what} has no forward-mode derivative")


def cache_append(cache: PagedCache, key: torch.Tensor, value: torch.Tensor, tables: torch.Tensor,
                 seq_lens: torch.Tensor, new_lens: Optional[torch.Tensor] = None) -> None:
    """Writes a batch's newest keys and values ``[B, L, H_kv, D]`` into ``cache``.

    ``seq_lens[b]`` counts the sample's tokens with the new ones: new token j is token
    ``t = seq_lens[b] - L + j``.  Tokens before a sequence's start (t < 0) are not
    written, nor, with ``new_lens``, any but the last ``new_lens[b]`` of the L: a batch of
    unlike numbers of new tokens is padded in front.  Token t goes to slot
    ``t % page_size`` of page ``tables[b, t // page_size]``; an entry outside
    ``[0, pages)``, such as -1, is no page and takes nothing.  The entries that a call
    writes to, of all samples, must name different pages (a table may name a page again
    where its tokens have left every window).  Cache tensors whose elements share memory,
    such as expanded ones, are refused.

    A page's and head's scale is the smallest power of two that brings the new tokens
    of the page to 448 at most, e4m3's largest value; where tokens of the page lie in
    front of them, at least the scale they have, and where it grows they are rescaled.
    Elements are rounded to the nearest, ties to even; NaN and infinities become NaN.

    float32, float16 or bfloat16, views of any strides; tables ``[B, M]``, ``seq_lens`` and
    ``new_lens`` int32 or int64.  Lengths on the device are taken as they are, clamped to
    ``[0, M * page_size]`` and ``[0, L]`` there; lengths on the host are checked and copied
    at every call, which waits for the stream; under graph capture they are refused.
    There is no derivative: inputs that require grad are refused outside
    ``torch.no_grad()``.
    """
    shape = _check_cache(cache)
    for t in cache:
        if not t.is_contiguous() and any(s == 0 and n > 1 for n, s in zip(t.shape, t.stride())):
            raise ValueError("cache_append cannot write to a cache whose elements share memory, got "
                             f"strides {[c.stride() for c in cache]}.")
    new = tuple(key.shape)
    if len(new) != 4 or value.shape != new or new[2:] != (shape[1], shape[3]):
        raise ValueError(f"key and value must be [B, L, {shape[1]}, {shape[3]}], got "
                         f"{tuple(key.shape)} and {tuple(value.shape)}.")
    if key.dtype != value.dtype:
        raise ValueError(f"key and value must have the same dtype, got {key.dtype} and {value.dtype}.")
    b, n = new[:2]
    _check_tables(tables, b, shape[2])
    _check_lens("seq_lens", seq_lens, b)
    capacity = tables.shape[1] * shape[2]
    if not seq_lens.is_cuda and key.is_cuda:
        seq_lens = _host_lens(seq_lens, capacity, key.device)
    if new_lens is not None:
        _check_lens("new_lens", new_lens, b)
        if not new_lens.is_cuda and key.is_cuda:
            new_lens = _host_lens(new_lens, n, key.device, "new_lens")
    op = None if _fused._py_autograd else _lib.node_op("cache_append", key, value)
    if op is not None:
        op(cache[0], cache[1], cache[2], cache[3], key, value, tables, seq_lens, new_lens,
           _lib.stream_of(key))
        return
    _no_derivative("cache_append", (key, value))
    hip.cache_append(cache, key, value, _narrow(tables, -1, 2 ** 31 - 1),
                     _narrow(seq_lens, 0, capacity),
                     None if new_lens is None else _narrow(new_lens, 0, n))


def cache_attention(query: torch.Tensor, cache: PagedCache, tables: torch.Tensor,
                    seq_lens: torch.Tensor, kernel_size: Optional[int] = None,
                    scale: Optional[float] = None, return_lse: bool = False
                    ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """The batch's newest tokens ``[B, L, H, D]`` (L = 1: one generated token each) attend
    to their samples' tokens in ``cache``, the new ones among them.

    ``seq_lens[b]`` counts the sample's tokens: query j is token ``t = seq_lens[b] - L + j``
    and sees the tokens up to t; with ``kernel_size`` the last ``kernel_size`` of them
    only, the causal window of ``na1d``.  Token i lies in slot ``i % page_size`` of page
    ``tables[b, i // page_size]``; tokens of an entry outside ``[0, pages)``, such as -1
    for pages that have left every window, are not seen.  What lies behind a length or
    in front of every window is not read.  A query that sees no key, such as one before
    the sequence's start (t < 0), or whose scores are all -inf, gets zeros and an LSE of
    -inf.

    float32, float16 or bfloat16 queries; query heads share key/value heads as in
    ``na1d``.  The cache's elements are taken exactly, and so are queries (in float32 to 24
    bits, to 2^-126 where they are smaller); products and sums are float32;
    probabilities are rounded to 16 bits for bfloat16 and float16 queries and to 24 for
    float32; sums may be divided differently, and differ in their last bits, for tables of
    another width or batches of other lengths.  Values are summed before the division, by
    weights of up to 2^8: 2^8 times a row's tokens times their largest value has to stay
    below 2^128.  The output has query's type; the LSE (``return_lse``) is float32
    ``[B, L, H]``, ready for ``merge_attentions``, as with ``prefix_attention`` over tokens
    that the batch shares.  ``tables`` and ``seq_lens`` as ``cache_append`` takes them.
    There is no derivative: inputs that require grad are refused outside
    ``torch.no_grad()``.
    """
    shape = _check_cache(cache)
    if query.ndim != 4 or query.shape[3] != shape[3]:
        raise ValueError(f"query must be [B, L, heads, {shape[3]}], got {tuple(query.shape)}.")
    b, _, h, d = query.shape
    if h < 1 or h % shape[1]:
        raise ValueError(f"heads_q ({h}) must be divisible by heads_kv ({shape[1]}) for GQA.")
    _check_tables(tables, b, shape[2])
    _check_lens("seq_lens", seq_lens, b)
    if kernel_size is not None and (not isinstance(kernel_size, int) or kernel_size < 1):
        raise ValueError(f"kernel_size must be a positive int or None, got {kernel_size!r}.")
    if scale is not None and not 2.0 ** -149 <= scale <= 2e38:  # (times log2 e a float32)
        raise ValueError(f"scale must be positive and at most 2e38, got {scale}.")
    capacity = tables.shape[1] * shape[2]
    scale = d ** -0.5 if scale is None else float(scale)
    if not seq_lens.is_cuda and query.is_cuda:
        seq_lens = _host_lens(seq_lens, capacity, query.device)
    window = 0 if kernel_size is None else kernel_size
    op = None if _fused._py_autograd else _lib.node_op("cache_attend", query, query)
    if op is not None:
        out, lse = op(query, cache[0], cache[1], cache[2], cache[3], tables, seq_lens, window, scale,
                      return_lse, _lib.stream_of(query))
    else:
        _no_derivative("cache_attention", (query,))
        out, lse = hip.cache_attend(query, cache, _narrow(tables, -1, 2 ** 31 - 1),
                                    _narrow(seq_lens, 0, capacity), window, scale, return_lse)
    return (out, lse) if return_lse else out


__all__ = ["PagedCache", "paged_cache", "cache_append", "cache_attention"]

# SPDX-License-Identifier: MIT OR Apache-2.0
"""A paged key-value cache: appending new tokens to it (rotated on the way) and attending over it.

The cache is two tensors of the caller's, `k_cache` and `v_cache`, [pages, page_size, key_heads, d]
in any order of the first three dims (a [pages, key_heads, page_size, d] pool is passed as its
transposed view), f32, f16 or bf16. `page_table` int32 [batch, width] gives the page of each
page_size rows of a sequence; entries past a sequence's length are not looked at. `lengths` int32
[batch] counts each sequence's keys, those of the current step included, so one tensor serves both
calls of a step:

    lengths += 1
    q = paged_append(k, v, k_cache, v_cache, page_table, lengths, q=q, freqs=freqs)
    o = paged_attention(q, k_cache, v_cache, page_table, lengths, scale)

Everything is read on the device when the kernels run: a captured CUDA graph of these lines can be
replayed while the lengths grow, up to the table's width. A page id outside the cache, or a length
past the table, raises `FusedAttentionError` on a later call (or in `check_status()`); the kernels
leave such keys out.
"""

from __future__ import annotations

import torch

from . import FusedAttentionError, _abi, _check_head_dim
from ._launch import (DTYPES, check_status, current_stream, int32_vector, merged_heads, no_gradient,
                      on_device, one_device, raise_if_expired, require)
from .positions import check_freqs

__all__ = ["paged_append", "paged_attention"]


def _check_cache(who, dtype, k_cache, v_cache, page_table, lengths, new_lengths, b, hk, d):
    shape = k_cache.shape
    if k_cache.dim() != 4 or v_cache.shape != shape or shape[2] != hk or shape[3] != d:
        raise FusedAttentionError(
            f"{who}: caches [pages, page_size, {hk}, {d}] expected, got {list(shape)} "
            f"{list(v_cache.shape)}")
    require(shape[1] >= 1, who, "a page needs at least one row")
    if k_cache.dtype not in DTYPES or v_cache.dtype != k_cache.dtype or (
            dtype != k_cache.dtype and dtype != torch.float32) or dtype not in DTYPES:
        raise FusedAttentionError(
            f"{who}: f32, f16 or bf16 inputs over a cache of their type, or f32 over any, expected; "
            f"got {dtype} over {k_cache.dtype} {v_cache.dtype}")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise FusedAttentionError(f"{who}: the caches' last dimension must be contiguous")
    if (page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.shape[0] != b
            or (page_table.shape[1] > 1 and page_table.stride(1) != 1)):
        raise FusedAttentionError(
            f"{who}: page_table int32 [{b}, width] with dense rows expected, got "
            f"{page_table.dtype} {list(page_table.shape)}")
    int32_vector(who, "lengths", lengths, b)
    int32_vector(who, "new_lengths", new_lengths, b)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [b, h, s, d] with its last dim contiguous."""
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def paged_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                 page_table: torch.Tensor, lengths: torch.Tensor, *,
                 q: torch.Tensor | None = None, freqs: torch.Tensor | None = None,
                 amplitude: float = 1.0, interleaved: bool = False,
                 new_lengths: torch.Tensor | None = None) -> torch.Tensor | None:
    """Writes new tokens' keys and values into the cache, in one launch; returns the rotated q.

    k, v [batch, key_heads, s, d] and q [batch, heads, s, d], any strides. Token i of a sequence's n
    new ones (n = s, or new_lengths[b] of a padded batch) sits at lengths[b] - n + i. With `freqs`
    (as for `rotary`) k and q are turned by that position; v and, without freqs, k and q are not.
    Values are rounded once to the cache's type. Padded rows of q come back as zeros; tokens without
    a page, and every other row of the cache, leave the cache as it was. Two tokens of a call must
    not have the same slot. -> q's rotation [batch, heads, s, d] (laid out as a dense [batch, s, heads,
    d]), or None without q. No gradients.
    """
    who = "paged_append"
    if k.dim() != 4 or v.shape != k.shape:
        raise FusedAttentionError(f"{who}: k and v [b, hk, s, d] expected, got {list(k.shape)} "
                                  f"{list(v.shape)}")
    b, hk, s, d = k.shape
    require(v.dtype == k.dtype, who, "k and v must have one type")
    if q is not None and (q.dim() != 4 or (q.shape[0], q.shape[2], q.shape[3]) != (b, s, d)
                          or q.dtype != k.dtype):
        raise FusedAttentionError(f"{who}: q [{b}, h, {s}, {d}] of k's type expected, got "
                                  f"{q.dtype} {list(q.shape)}")
    _check_cache(who, k.dtype, k_cache, v_cache, page_table, lengths, new_lengths, b, hk, d)
    dev = one_device(who, k, v, k_cache, v_cache, page_table, lengths, new_lengths, q, freqs)
    no_gradient(who, q, k, v, k_cache, v_cache)
    if freqs is not None:
        check_freqs(who, freqs, d)
    raise_if_expired()
    k, v = _rows(k), _rows(v)
    out, h = None, 0
    if q is not None:
        q, h = _rows(q), q.shape[1]
        out = merged_heads(b, h, s, d, q)
    with on_device(dev):
        st = _abi.paged_append(
            None if q is None else q.data_ptr(), None if q is None else q.stride()[:3],
            None if q is None else out.data_ptr(), None if q is None else (s * h * d, d, h * d),
            k.data_ptr(), k.stride()[:3], v.data_ptr(), v.stride()[:3], DTYPES[k.dtype],
            k_cache.data_ptr(), k_cache.stride()[:3], v_cache.data_ptr(), v_cache.stride()[:3],
            DTYPES[k_cache.dtype], k_cache.shape[0], k_cache.shape[1], page_table.data_ptr(),
            page_table.stride(0), page_table.shape[1], lengths.data_ptr(),
            None if new_lengths is None else new_lengths.data_ptr(),
            None if freqs is None else freqs.data_ptr(), float(amplitude), b, h, hk, s, d,
            0 if freqs is None else 2 * freqs.numel(), interleaved, current_stream(dev))
    check_status(st, who)
    return out


def _aligned(t: torch.Tensor) -> bool:
    unit = 16 // t.element_size()
    st = t.stride()
    return (t.data_ptr() % 16 == 0 and st[3] == 1 and st[0] % unit == 0 and st[1] % unit == 0
            and st[2] % unit == 0)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                    new_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's newest s tokens (one, or a few) over its cached keys.

    q [batch, heads, s, d], d in HEAD_DIMS, of the cache's type or f32; heads a multiple of the
    cache's key heads. Query i of a sequence's n (n = s, or new_lengths[b]) sees its first
    lengths[b] - n + i + 1 keys: all of them for a single token. The cache's rows must be 16-byte
    aligned. -> [batch, heads, s, d], laid out as a dense [batch, s, heads, d], of q's type; zeros
    where a query sees no key or a padded row is no query. The keys are split into chunks by the
    sequence's own length and joined in order: bit-identical across reruns and batches. Softmax
    statistics and sums are fp32. No gradients.
    """
    who = "paged_attention"
    require(q.dim() == 4, who, f"q [b, h, s, d] expected, shape {list(q.shape)}")
    b, h, s, d = q.shape
    _check_head_dim(d)
    hk = k_cache.shape[2] if k_cache.dim() == 4 else 0
    _check_cache(who, q.dtype, k_cache, v_cache, page_table, lengths, new_lengths, b, hk, d)
    if (h % hk if hk else h) != 0:
        raise FusedAttentionError(f"{who}: {h} query heads are no multiple of {hk} key heads")
    dev = one_device(who, q, k_cache, v_cache, page_table, lengths, new_lengths)
    no_gradient(who, q, k_cache, v_cache)
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        require(_aligned(t) or t.numel() == 0, who, f"{name}: rows must be 16-byte aligned")
    raise_if_expired()
    if not _aligned(q):
        q = q.clone(memory_format=torch.contiguous_format)
    o = merged_heads(b, h, s, d, q)
    width, page = page_table.shape[1], k_cache.shape[1]
    n = _abi.paged_attention_workspace_bytes(b, h, s, width * page, d, DTYPES[k_cache.dtype])
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    with on_device(dev):
        st = _abi.paged_attention(
            q.data_ptr(), q.stride()[:3], DTYPES[q.dtype], k_cache.data_ptr(), k_cache.stride()[:3],
            v_cache.data_ptr(), v_cache.stride()[:3], DTYPES[k_cache.dtype], k_cache.shape[0], page,
            page_table.data_ptr(), page_table.stride(0), width, lengths.data_ptr(),
            None if new_lengths is None else new_lengths.data_ptr(), o.data_ptr(),
            None if ws is None else ws.data_ptr(), n, b, h, hk, s, d, float(scale), current_stream(dev))
    check_status(st, who)
    return o

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
replayed while the lengths grow, up to the table's width. Where a page id lies outside the cache, or
a length past the table, the kernels leave such keys out and go on; `check_status()` raises
`FusedAttentionError` for it, and no other call does (it may serve another sequence).
"""

from __future__ import annotations

import torch

from ._binding import _ops

__all__ = ["paged_append", "paged_attention"]


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
    return _ops.paged_append(k, v, k_cache, v_cache, page_table, lengths, q, freqs, amplitude,
                             interleaved, new_lengths)


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    page_table: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                    new_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's newest s tokens (one, or a few) over its cached keys.

    q [batch, heads, s, d], d in HEAD_DIMS, of the cache's type or f32; heads a multiple of the
    cache's key heads. Query i of a sequence's n (n = s, or new_lengths[b]) sees its first
    lengths[b] - n + i + 1 keys: all of them for a single token. The cache's rows must be 16-byte
    aligned. -> [batch, heads, s, d], laid out as a dense [batch, s, heads, d], of q's type; zeros
    where a query sees no key or a padded row is no query. What a query sees is to be finite (with an
    infinity the result may be NaN where the formula has a value, in its own sequence; what none sees
    may be anything).
    The keys are split into chunks by the
    sequence's own length and joined in order: bit-identical across reruns and batches. Softmax
    statistics and sums are fp32. No gradients.
    """
    return _ops.paged_attention(q, k_cache, v_cache, page_table, lengths, scale, new_lengths)

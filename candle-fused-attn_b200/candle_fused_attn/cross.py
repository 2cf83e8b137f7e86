# SPDX-License-Identifier: MIT OR Apache-2.0
"""Attention to another sequence's states (an encoder's): queries and keys of different lengths, a
padded batch of keys, key heads shared by groups of query heads; fp32, with gradients."""

from __future__ import annotations

import torch

from ._binding import _ops

__all__ = ["cross_attention"]


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                    key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v of queries over another sequence's keys and values.

    q [batch, heads, sq, d], k and v [batch, key_heads, sk, d], f32 on CUDA, d in HEAD_DIMS, any
    strides (rows that are not 16-byte aligned are copied first); heads a multiple of key_heads:
    query head i reads key head i // (heads // key_heads). `key_lengths`: int32 [batch] on the
    device, how many keys each batch element has (values are held within 0 .. sk); what lies behind
    them is not read into any result, and a query without a key gives zeros and no gradient. What a
    query does see is to be finite (operands enter the tensor cores in parts, and with an infinity the
    result may be NaN where the formula has a value, in its own batch element).
    -> [batch, heads, sq, d], laid out as a dense [batch, sq, heads, d].

    Differentiable in q, k and v (dk, dv of a shared head are summed over its query heads). Few
    queries -- the single token of a decoding step -- take a kernel that splits the keys.
    The backward asks for up to 4 GB of scratch beside its gradients and goes on, with the same bits
    but slower, where that cannot be had. Bit-identical across reruns and batch splits.
    """
    return _ops.cross_attention(q, k, v, scale, key_lengths)

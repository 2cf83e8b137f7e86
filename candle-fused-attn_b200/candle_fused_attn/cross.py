# SPDX-License-Identifier: MIT OR Apache-2.0
"""Attention to another sequence's states (an encoder's): queries and keys of different lengths, a
padded batch of keys, key heads shared by groups of query heads; fp32, with gradients."""

from __future__ import annotations

import torch

from . import FusedAttentionError, _abi, _check_head_dim, _float4_rows
from ._launch import (check_status, current_stream, first_order, int32_vector, merged_heads,
                      on_device, one_device, raise_if_expired, require)

__all__ = ["cross_attention"]

# Up to as many query rows a key head (query heads of a group x queries) the forward without gradients
# runs split over the keys, one block a chunk of keys and up to 16 rows; above, the tensor-core kernels,
# which take 256 rows a block. The batch plays no part: the choice changes bits. Split and whole, in us,
# [b, 6, rows, 64] over 1500 keys: 16 rows 11 and 55 (b 1), 23 and 58 (16), 82 and 169 (64); 32 rows 11
# and 55, 42 and 58, 156 and 169; 48 rows 11 and 55, 60 and 58, 226 and 170.
FEW_ROWS = 32


def _dims(q, k, v):
    if (q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0]
            or k.shape[3] != q.shape[3]):
        raise FusedAttentionError(
            "cross_attention: q [b, h, sq, d], k and v [b, hk, sk, d] expected, got "
            f"{list(q.shape)} {list(k.shape)} {list(v.shape)}")
    (b, h, sq, d), (hk, sk) = q.shape, k.shape[1:3]
    if (h % hk if hk else h) != 0:
        raise FusedAttentionError(
            f"cross_attention: {h} query heads are no multiple of {hk} key heads")
    _check_head_dim(d)
    return b, h, hk, sq, sk, d


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


def _forward(q, k, v, key_lengths, scale, dims):
    b, h, hk, sq, sk, d = dims
    dev = q.device
    raise_if_expired()
    o = merged_heads(b, h, sq, d, q)
    lse = torch.empty((b, h, sq), dtype=torch.float32, device=dev)
    with on_device(dev):
        st = _abi.cross_fwd(q.data_ptr(), q.stride()[:3], k.data_ptr(), k.stride()[:3],
                            v.data_ptr(), v.stride()[:3], _ptr(key_lengths), o.data_ptr(),
                            lse.data_ptr(), b, h, hk, sq, sk, d, scale, current_stream(dev))
    check_status(st, "cross_attention")
    return o, lse


def _few(q, k, v, key_lengths, scale, dims):
    b, h, hk, sq, sk, d = dims
    dev = q.device
    raise_if_expired()
    o = merged_heads(b, h, sq, d, q)
    n = _abi.cross_few_workspace_bytes(b, h, sq, sk, d)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    with on_device(dev):
        st = _abi.cross_few(q.data_ptr(), q.stride()[:3], k.data_ptr(), k.stride()[:3],
                            v.data_ptr(), v.stride()[:3], _ptr(key_lengths), o.data_ptr(),
                            _ptr(ws), n, b, h, hk, sq, sk, d, scale, current_stream(dev))
    check_status(st, "cross_attention")
    return o


class _CrossAttention(torch.autograd.Function):
    """q [b, h, sq, d], k and v [b, hk, sk, d] -> [b, h, sq, d]."""

    @staticmethod
    def forward(ctx, q, k, v, key_lengths, scale, dims):
        o, lse = _forward(q, k, v, key_lengths, scale, dims)
        ctx.save_for_backward(q, k, v, key_lengths, o, lse)
        ctx.scale, ctx.dims = scale, dims
        return o

    @staticmethod
    @first_order
    def backward(ctx, grad):
        q, k, v, key_lengths, o, lse = ctx.saved_tensors
        b, h, hk, sq, sk, d = ctx.dims
        dev = q.device
        raise_if_expired()
        grad = _float4_rows(grad)
        dq = merged_heads(b, h, sq, d, q)
        dkv = torch.empty((b, sk, 2, hk, d), dtype=torch.float32, device=dev)
        n = _abi.cross_bwd_workspace_bytes_fast(b, h, hk, sq, sk, d)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        with on_device(dev):
            st = _abi.cross_bwd(q.data_ptr(), q.stride()[:3], k.data_ptr(), k.stride()[:3],
                                v.data_ptr(), v.stride()[:3], _ptr(key_lengths), o.data_ptr(),
                                lse.data_ptr(), grad.data_ptr(), grad.stride()[:3], dq.data_ptr(),
                                dkv.data_ptr(), ws.data_ptr(), n, b, h, hk, sq, sk, d, ctx.scale,
                                current_stream(dev))
        check_status(st, "cross_attention")
        shape, strides = (b, hk, sk, d), (2 * sk * hk * d, d, 2 * hk * d, 1)
        return (dq, dkv.as_strided(shape, strides), dkv.as_strided(shape, strides, hk * d),
                None, None, None)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float,
                    key_lengths: torch.Tensor | None = None) -> torch.Tensor:
    """softmax(q k^T scale) v of queries over another sequence's keys and values.

    q [batch, heads, sq, d], k and v [batch, key_heads, sk, d], f32 on CUDA, d in HEAD_DIMS, any
    strides (rows that are not 16-byte aligned are copied first); heads a multiple of key_heads:
    query head i reads key head i // (heads // key_heads). `key_lengths`: int32 [batch] on the
    device, how many keys each batch element has (values are held within 0 .. sk); what lies behind
    them is not read into any result, and a query without a key gives zeros and no gradient.
    -> [batch, heads, sq, d], laid out as a dense [batch, sq, heads, d].

    Differentiable in q, k and v (dk, dv of a shared head are summed over its query heads). Without
    gradients, few queries -- the single token of a decoding step -- take a kernel that splits the
    keys instead. Bit-identical across reruns and batch splits.
    """
    q, k, v = (_float4_rows(t) if t.dim() == 4 else t for t in (q, k, v))
    for t in (q, k, v):
        require(t.dtype == torch.float32, "cross_attention", "f32 only")
    dims = _dims(q, k, v)
    one_device("cross_attention", q, k, v, key_lengths)
    int32_vector("cross_attention", "key_lengths", key_lengths, dims[0])
    scale = float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _CrossAttention.apply(q, k, v, key_lengths, scale, dims)
    if dims[2] and dims[1] // dims[2] * dims[3] <= FEW_ROWS:
        return _few(q, k, v, key_lengths, scale, dims)
    return _forward(q, k, v, key_lengths, scale, dims)[0]

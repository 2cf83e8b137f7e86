# SPDX-License-Identifier: MIT OR Apache-2.0
"""What the operators beside the fused attention share: argument checks, the current device and
stream, and status codes as errors."""

from __future__ import annotations

import contextlib

import torch
from torch.autograd.function import once_differentiable

from . import FusedAttentionError, _abi, _raise_if_expired, _sink_flag, _stream

DTYPES = {torch.float32: _abi.CFA_F32, torch.float16: _abi.CFA_F16, torch.bfloat16: _abi.CFA_BF16}
_nothing = contextlib.nullcontext()


def require(ok: bool, who: str, what: str) -> None:
    if not ok:
        raise FusedAttentionError(f"{who}: {what}")


def one_device(who: str, *ts: torch.Tensor | None) -> torch.device:
    """The CUDA device that every given tensor is on."""
    index = ts[0].get_device()
    for t in ts:
        if t is not None and (t.get_device() != index or index < 0):
            if not all(x is None or x.is_cuda for x in ts):
                raise FusedAttentionError(f"{who}: CUDA tensors required")
            raise FusedAttentionError(f"{who}: tensors on different devices")
    return ts[0].device


def merged_heads(b: int, h: int, s: int, d: int, like: torch.Tensor) -> torch.Tensor:
    """An empty [b, h, s, d] tensor laid out as [b, s, h, d] (merge-heads ready), of like's type."""
    return torch.empty_strided((b, h, s, d), (s * h * d, d, h * d, 1), dtype=like.dtype,
                               device=like.device)


def int32_vector(who: str, name: str, t: torch.Tensor | None, n: int) -> None:
    if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n
                          or (n > 1 and t.stride(0) != 1)):
        raise FusedAttentionError(
            f"{who}: {name} must be a dense int32 tensor [{n}], got {t.dtype} {list(t.shape)}")


def no_gradient(who: str, *ts: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise FusedAttentionError(f"{who}: has no backward (call it under torch.no_grad())")


# (torch.cuda.current_stream builds a Stream object to read one integer of: 2 us of a 10 us call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def current_stream(dev: torch.device) -> int:
    """The current stream of `dev` as the handle that the ABI takes."""
    return _stream(dev) if _raw_stream is None else _raw_stream(dev.index)


def on_device(dev: torch.device):
    """The device as the current one for a launch (free where it is already)."""
    return _nothing if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def check_status(status: int, who: str) -> None:
    if status != _abi.CFA_OK:
        raise FusedAttentionError(f"{who}: {_abi.strerror(status)}")


def first_order(backward):
    """A Function's backward whose result cannot be differentiated again: an error then. (The wrapper that
    watches for it costs 10 us, and only `create_graph` needs it.)"""
    watched = once_differentiable(backward)

    def call(ctx, grad):
        return (watched if torch.is_grad_enabled() else backward)(ctx, grad)

    return call


_flag = None


def raise_if_expired() -> None:
    """As the fused attention does before a launch (its check, without looking the flag up each time)."""
    global _flag
    if _flag is None:
        _flag = _sink_flag()
    if _flag.value:
        _raise_if_expired()

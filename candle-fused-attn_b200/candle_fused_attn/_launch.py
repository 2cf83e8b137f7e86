# SPDX-License-Identifier: MIT OR Apache-2.0
"""What the operators beside the fused attention share: argument checks, the current device and
stream, and status codes as errors."""

from __future__ import annotations

import contextlib

import torch

from . import FusedAttentionError, _abi, _raise_if_expired

DTYPES = {torch.float32: _abi.CFA_F32, torch.float16: _abi.CFA_F16, torch.bfloat16: _abi.CFA_BF16}
_nothing = contextlib.nullcontext()


def require(ok: bool, who: str, what: str) -> None:
    if not ok:
        raise FusedAttentionError(f"{who}: {what}")


def one_device(who: str, *ts: torch.Tensor | None) -> torch.device:
    """The CUDA device that every given tensor is on."""
    dev = ts[0].device
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise FusedAttentionError(f"{who}: CUDA tensors required")
        if t.device != dev:
            raise FusedAttentionError(f"{who}: tensors on different devices")
    return dev


def int32_vector(who: str, name: str, t: torch.Tensor | None, n: int) -> None:
    if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != n
                          or (n > 1 and t.stride(0) != 1)):
        raise FusedAttentionError(
            f"{who}: {name} must be a dense int32 tensor [{n}], got {t.dtype} {list(t.shape)}")


def no_gradient(who: str, *ts: torch.Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise FusedAttentionError(f"{who}: has no backward (call it under torch.no_grad())")


def on_device(dev: torch.device):
    """The device as the current one for a launch (free where it is already)."""
    return _nothing if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def check_status(status: int, who: str) -> None:
    if status != _abi.CFA_OK:
        raise FusedAttentionError(f"{who}: {_abi.strerror(status)}")


raise_if_expired = _raise_if_expired

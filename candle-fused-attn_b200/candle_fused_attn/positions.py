# SPDX-License-Identifier: MIT OR Apache-2.0
"""Rotary positions for queries and keys, between the projection and the attention."""

from __future__ import annotations

import math

import torch

from . import FusedAttentionError, _abi, qkv_geometry
from ._launch import (DTYPES, check_status, current_stream, first_order, merged_heads, no_gradient,
                      on_device, one_device, raise_if_expired, require)

__all__ = ["rotary", "rotary_qkv", "rotary_frequencies"]


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str | None = None,
                       factor: float = 1.0, original_length: int | None = None,
                       beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str = "cuda") -> tuple[torch.Tensor, float]:
    """The `freqs` and `amplitude` of `rotary`: f_j = base^(-2j / rotary_dim) radians a position,
    j < rotary_dim / 2, as a float64 tensor, and 1.0; for contexts `factor` times longer:

    - "linear": f_j / factor (positions pressed together);
    - "ntk": base * factor^(rotary_dim / (rotary_dim - 2)) (the slowest frequency divided by factor,
      the fastest left alone);
    - "yarn": by the turns a frequency makes over `original_length` positions: above beta_fast as it
      is, below beta_slow divided by factor, linear in the turns between; amplitude
      0.1 ln(factor) + 1.
    """
    who = "rotary_frequencies"
    require(rotary_dim > 0 and rotary_dim % 2 == 0, who,
            f"an even rotary dimension expected, got {rotary_dim}")
    require(base > 0 and factor > 0, who, "base and factor must be positive")
    j = torch.arange(rotary_dim // 2, dtype=torch.float64)
    amplitude = 1.0
    if scaling == "ntk" and rotary_dim > 2:
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    freqs = float(base) ** (-2.0 * j / rotary_dim)
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        require(original_length is not None and original_length > 0, who,
                "yarn scaling needs original_length")
        require(beta_fast > beta_slow, who, "beta_fast must exceed beta_slow")
        turns = original_length * freqs / (2 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        freqs = freqs * keep + freqs / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise FusedAttentionError(f"{who}: unknown scaling {scaling!r} (linear, ntk or yarn)")
    return freqs.to(device), amplitude


def check_freqs(who: str, freqs: torch.Tensor, d: int) -> None:
    no_gradient(f"{who}: freqs", freqs)
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or (freqs.numel() > 1
                                                            and freqs.stride(0) != 1):
        raise FusedAttentionError(
            f"{who}: freqs must be a dense float64 vector, got {freqs.dtype} {list(freqs.shape)}")
    if 2 * freqs.numel() > d:
        raise FusedAttentionError(
            f"{who}: {freqs.numel()} frequencies turn {2 * freqs.numel()} dims, the head has {d}")


def _launch(who, x_ptr, xs, dtype, dims, rotated, positions, freqs, amplitude, interleaved, inverse,
            out, outs, dev):
    """One cfa_rotary call over [b, h, s, d]; positions: an int or a [b, s] tensor."""
    b, h, s, d = dims
    raise_if_expired()
    at = (None, 0, None, positions) if isinstance(positions, int) else (
        positions.data_ptr(), positions.element_size(), positions.stride(), 0)
    with on_device(dev):
        st = _abi.rotary(x_ptr, xs, out.data_ptr(), outs, DTYPES[dtype], *at, freqs.data_ptr(),
                         amplitude, b, h, rotated, s, d, 2 * freqs.numel(), interleaved, inverse,
                         current_stream(dev))
    check_status(st, who)


def _turn(x, positions, freqs, amplitude, interleaved, inverse):
    b, h, s, d = x.shape
    if x.stride(3) != 1 and d > 1:
        x = x.contiguous()
    y = merged_heads(b, h, s, d, x)
    _launch("rotary", x.data_ptr(), x.stride()[:3], x.dtype, (b, h, s, d), h, positions, freqs,
            amplitude, interleaved, inverse, y, (s * h * d, d, h * d), x.device)
    return y


class _Rotary(torch.autograd.Function):
    """y = R x; dx = R^T dy, the inverse rotation with the same amplitude."""

    @staticmethod
    def forward(ctx, x, positions, freqs, amplitude, interleaved):
        ctx.save_for_backward(freqs, *(() if isinstance(positions, int) else (positions,)))
        ctx.first = positions if isinstance(positions, int) else None
        ctx.amplitude, ctx.interleaved = amplitude, interleaved
        return _turn(x, positions, freqs, amplitude, interleaved, False)

    @staticmethod
    @first_order
    def backward(ctx, grad):
        freqs, *at = ctx.saved_tensors
        positions = at[0] if at else ctx.first
        dx = _turn(grad, positions, freqs, ctx.amplitude, ctx.interleaved, True)
        return dx, None, None, None, None


def _turn_qkv(qkv, heads, positions, freqs, amplitude, interleaved, inverse):
    if qkv.stride(2) != 1:
        qkv = qkv.contiguous()
    (b, h, s, d), strides, _ = qkv_geometry(tuple(qkv.shape), qkv.stride(), heads)
    out = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
    _launch("rotary_qkv", qkv.data_ptr(), strides, qkv.dtype, (b, 3 * h, s, d), 2 * h, positions,
            freqs, amplitude, interleaved, inverse, out, (s * 3 * h * d, d, 3 * h * d), qkv.device)
    return out


class _RotaryQkv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, heads, positions, freqs, amplitude, interleaved):
        ctx.save_for_backward(freqs, *(() if isinstance(positions, int) else (positions,)))
        ctx.first = positions if isinstance(positions, int) else None
        ctx.heads, ctx.amplitude, ctx.interleaved = heads, amplitude, interleaved
        return _turn_qkv(qkv, heads, positions, freqs, amplitude, interleaved, False)

    @staticmethod
    @first_order
    def backward(ctx, grad):
        freqs, *at = ctx.saved_tensors
        positions = at[0] if at else ctx.first
        d = _turn_qkv(grad, ctx.heads, positions, freqs, ctx.amplitude, ctx.interleaved, True)
        return d, None, None, None, None, None


def _check(who, x, positions, freqs, b, s, d):
    if x.dtype not in DTYPES:
        raise FusedAttentionError(f"{who}: f32, f16 or bf16 expected, got {x.dtype}")
    check_freqs(who, freqs, d)
    if isinstance(positions, torch.Tensor):
        one_device(who, x, freqs, positions)
        if positions.dtype not in (torch.int32, torch.int64):
            raise FusedAttentionError(f"{who}: int32 or int64 positions expected")
        if positions.dim() > 2 or positions.shape not in ((s,), (b, s), (1, s), (b, 1)):
            raise FusedAttentionError(f"{who}: positions [{s}] or [{b}, {s}] expected, got "
                                      f"{list(positions.shape)}")
        return positions if positions.shape == (b, s) else positions.expand(b, s)
    one_device(who, x, freqs)
    return int(positions)


def rotary(x: torch.Tensor, positions: torch.Tensor | int, freqs: torch.Tensor, *,
           amplitude: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """x with each head's first 2 len(freqs) dims turned by its position.

    x [batch, heads, seq, d] (queries or keys), f32, f16 or bf16 on CUDA, any strides, d <= 1024.
    `positions`: int32 or int64 [seq] or [batch, seq] on the device, or the first position (an int)
    of consecutive ones. `freqs`: float64 radians a position (`rotary_frequencies`); pair j is
    (j, j + len(freqs)), or (2j, 2j + 1) with `interleaved`, and is turned by position * freqs[j] and
    scaled by `amplitude`; the dims past the pairs are copied. Angles are reduced in 64 bits, so far
    positions lose nothing. -> [batch, heads, seq, d], laid out as a dense [batch, seq, heads, d], of
    x's type. Differentiable in x.
    """
    require(x.dim() == 4, "rotary", f"[b, h, s, d] expected, shape {list(x.shape)}")
    b, _, s, d = x.shape
    at = _check("rotary", x, positions, freqs, b, s, d)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Rotary.apply(x, at, freqs, float(amplitude), bool(interleaved))
    return _turn(x, at, freqs, float(amplitude), bool(interleaved), False)


def rotary_qkv(qkv: torch.Tensor, heads: int, positions: torch.Tensor | int, freqs: torch.Tensor, *,
               amplitude: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """`rotary` on the queries and keys of a fused projection [batch, seq, 3 heads d] (the values are
    copied): what `fused_attention_qkv` then takes. One launch, one gradient laid out like `qkv`."""
    (b, h, s, d), _, _ = qkv_geometry(tuple(qkv.shape), (0, 0, 1), int(heads))
    at = _check("rotary_qkv", qkv, positions, freqs, b, s, d)
    args = (qkv, h, at, freqs, float(amplitude), bool(interleaved))
    if torch.is_grad_enabled() and qkv.requires_grad:
        return _RotaryQkv.apply(*args)
    return _turn_qkv(*args, False)

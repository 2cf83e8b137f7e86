# SPDX-License-Identifier: MIT OR Apache-2.0
"""Rotary positions for queries and keys, between the projection and the attention."""

from __future__ import annotations

import math

import torch

from . import FusedAttentionError
from ._binding import _ops, require

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
      0.1 ln(factor) + 1. (A model trained with a ramp over the index j between rounded bounds has
      other frequencies in between: pass its own as `freqs`.)
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


def rotary(x: torch.Tensor, positions: torch.Tensor | int, freqs: torch.Tensor, *,
           amplitude: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """x with each head's first 2 len(freqs) dims turned by its position.

    x [batch, heads, seq, d] (queries or keys), f32, f16 or bf16 on CUDA, any strides, d <= 1024.
    `positions`: int32 or int64 on the device, one a token ([seq] or [batch, seq]) or one for all of
    a sequence's tokens ([batch, 1]: not the first of consecutive ones); or an int, the first of
    consecutive ones. `freqs`: float64 radians a position (`rotary_frequencies`); pair j is
    (j, j + len(freqs)), or (2j, 2j + 1) with `interleaved`, and is turned by position * freqs[j] and
    scaled by `amplitude`; the dims past the pairs are copied. Angles are reduced in 64 bits, so far
    positions lose nothing. -> [batch, heads, seq, d], laid out as a dense [batch, seq, heads, d], of
    x's type. Differentiable in x.
    """
    return _ops.rotary(x, positions, freqs, amplitude, interleaved)


def rotary_qkv(qkv: torch.Tensor, heads: int, positions: torch.Tensor | int, freqs: torch.Tensor, *,
               amplitude: float = 1.0, interleaved: bool = False) -> torch.Tensor:
    """`rotary` on the queries and keys of a fused projection [batch, seq, 3 heads d] (the values are
    copied): what `fused_attention_qkv` then takes. One launch, one gradient laid out like `qkv`."""
    return _ops.rotary_qkv(qkv, heads, positions, freqs, amplitude, interleaved)

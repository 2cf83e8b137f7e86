# SPDX-License-Identifier: MIT OR Apache-2.0
"""Arguments that the operators refuse, on the CPU (before a device is looked at)."""

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi


@pytest.mark.parametrize("shape", [(3, 4), (3, 1), (2, 3), (5,), (1,), (1, 2, 4), ()])
def test_positions_of_other_shapes(shape):
    x, f = torch.zeros(2, 3, 4, 8), torch.ones(4, dtype=torch.float64)
    at = torch.zeros(shape, dtype=torch.int64)
    for call in (lambda: cfa.rotary(x, at, f), lambda: cfa.rotary_qkv(torch.zeros(2, 4, 72), 3, at, f)):
        with pytest.raises(cfa.FusedAttentionError, match=r"positions \[4\], \[2, 4\] or \[2, 1\] expected"):
            call()


@pytest.mark.parametrize("shape", [(4,), (2, 4), (1, 4), (2, 1)])
def test_positions_that_are_taken(shape):
    """One a token, or a sequence's one for all of its tokens."""
    x, f = torch.zeros(2, 3, 4, 8), torch.ones(4, dtype=torch.float64)
    with pytest.raises(cfa.FusedAttentionError, match="CUDA tensors required"):
        cfa.rotary(x, torch.zeros(shape, dtype=torch.int32), f)


def test_cross_backward_parts_are_bounded():
    """[b, 16 over 1, 1024 x 1024, 64]: 8 key blocks of one key head over 256 query tiles, 19 parts with a dK
    and dV of their own, of 0.5 MB each. Up to 512 MB of them, whatever the batch."""
    size, each = _abi.cross_bwd_workspace_bytes, 19 * 1024 * 2 * 64 * 4
    for b in (1, 2, 53, 54, 64, 1024):
        rest = 256 + b * 256 * 4 + b * 16 * 1024 * 4  # ticket, turn counters, D
        slices = min(b, (512 << 20) // each)
        assert slices * each + rest <= size(b, 16, 1, 1024, 1024, 64) <= slices * each + rest + 1024

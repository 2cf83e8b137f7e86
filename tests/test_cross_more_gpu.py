# SPDX-License-Identifier: MIT OR Apache-2.0
"""Cross attention at the sizes and scales that tests/test_cross_gpu.py leaves out; its band."""

import pytest
import torch

import candle_fused_attn as cfa
from test_cross_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sk", [1, 15, 16, 17, 33, 48, 63, 65, 127])
def test_few_query_rows_over_few_keys(cuda, d, sk):
    """Fewer keys than the four warps of a block take at once: some leave at their first tile, while the
    copies of their second are on the way."""
    for h, hk, sq in ((2, 2, 5), (4, 1, 4), (3, 1, 10)):
        check(cuda, 3, h, hk, sq, sk, d, [sk, 0, (sk + 1) // 2], seed=sk)
    cfa.check_status()

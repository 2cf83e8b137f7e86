# SPDX-License-Identifier: MIT OR Apache-2.0
"""A bad page id is data of one sequence: it is reported, and fails nobody else's call."""

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi

FAKE = 1 << 20


def test_page_sink_host_checks():
    """As cfa_error_sink's: NULL unregisters, a misaligned address is refused before any CUDA call."""
    assert _abi.page_sink(None) == _abi.CFA_OK
    assert _abi.page_sink(FAKE + 2) == _abi.CFA_ERR_ALIGNMENT
    assert _abi.page_sink(None) == _abi.CFA_OK


def requests(cuda):
    """Two sequences of 20 keys; the second one's last page is no page of the cache."""
    kc, vc = torch.randn(2, 4, 16, 2, 64, device=cuda)
    table = torch.tensor([[0, 1], [2, 1000]], dtype=torch.int32, device=cuda)
    lengths = torch.tensor([20, 20], dtype=torch.int32, device=cuda)
    return torch.randn(2, 2, 1, 64, device=cuda), kc, vc, table, lengths


@pytest.mark.gpu
@pytest.mark.parametrize("by", ["attention", "append"])
def test_other_calls_go_on(cuda, by):
    q, kc, vc, table, lengths = requests(cuda)
    good = (q[:1], kc, vc, table[:1], lengths[:1])
    want = cfa.paged_attention(*good, 0.125)
    x = torch.randn(1, 2, 40, 64, device=cuda, requires_grad=True)
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    cfa.check_status()
    if by == "attention":
        both = cfa.paged_attention(q, kc, vc, table, lengths, 0.125)
        assert torch.equal(both[:1], want)
    else:
        cfa.paged_append(q, q, kc.clone(), vc.clone(), table, lengths)
    torch.cuda.synchronize()
    assert torch.equal(cfa.paged_attention(*good, 0.125), want)
    cfa.paged_append(q[:1], q[:1], kc.clone(), vc.clone(), table[:1], lengths[:1])
    for y in (cfa.rotary(x, 0, freqs), cfa.cross_attention(x, x, x, 0.125), cfa.fused_attention(x, x, x, 0.125, False)):
        torch.autograd.grad(y.sum(), x)
    with pytest.raises(cfa.FusedAttentionError, match="page id"):
        cfa.check_status()
    cfa.check_status()  # reported once


@pytest.mark.gpu
def test_a_bad_page_does_not_cover_an_expired_wait(cuda):
    """A bounded wait that expires (results invalid) and, behind it, a bad page: the next call raises for the
    one, check_status() for the other."""
    q, kc, vc, table, lengths = requests(cuda)
    cfa.paged_attention(q[:1], kc, vc, table[:1], lengths[:1], 0.125)
    cfa.check_status()
    ws = torch.zeros(256, dtype=torch.uint8, device=cuda)
    assert _abi.selftest_bounded_wait(ws.data_ptr(), 20_000_000, 2, torch.cuda.current_stream().cuda_stream) == _abi.CFA_OK
    cfa.paged_attention(q, kc, vc, table, lengths, 0.125)
    torch.cuda.synchronize()
    with pytest.raises(cfa.FusedAttentionError, match="expired"):
        cfa.paged_attention(q[:1], kc, vc, table[:1], lengths[:1], 0.125)
    with pytest.raises(cfa.FusedAttentionError, match="page id"):
        cfa.check_status()
    cfa.check_status()

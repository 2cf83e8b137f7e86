# SPDX-License-Identifier: MIT OR Apache-2.0
"""Cross attention at the sizes and scales that tests/test_cross_gpu.py leaves out; its band."""

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi
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


@pytest.mark.parametrize("d,b,h,sq,sk", [(64, 60, 16, 1024, 1024), (128, 120, 8, 512, 600), (32, 200, 16, 600, 700)])
def test_a_batch_whose_parts_take_slices(cuda, d, b, h, sq, sk):
    """More than 512 MB of the parts' dK and dV: the batch goes in slices. Each element's gradients are those it
    has alone, bit for bit, with the partials of dQ and (the least workspace) by the turn chain."""
    g = torch.Generator(device=cuda).manual_seed(d)
    q, dout = (torch.randn(b, h, sq, d, device=cuda, generator=g) for _ in range(2))
    k, v = (torch.randn(b, 1, sk, d, device=cuda, generator=g) for _ in range(2))
    lengths = torch.full((b,), sk, dtype=torch.int32, device=cuda)
    lengths[1::3], lengths[7] = sk // 2 + 3, 0
    alone = _abi.cross_bwd_workspace_bytes(1, h, 1, sq, sk, d)
    assert _abi.cross_bwd_workspace_bytes(b, h, 1, sq, sk, d) < 0.95 * b * alone
    x = [t.requires_grad_(True) for t in (q, k, v)]
    o = cfa.cross_attention(*x, 0.1, key_lengths=lengths)
    grads = torch.autograd.grad(o, x, dout)
    for i in (0, 1, 7, b // 2, b - 2, b - 1):
        y = [t[i:i + 1].detach().requires_grad_(True) for t in x]
        oi = cfa.cross_attention(*y, 0.1, key_lengths=lengths[i:i + 1])
        gi = torch.autograd.grad(oi, y, dout[i:i + 1])
        assert torch.equal(oi[0], o[i]) and all(torch.equal(a[0], c[i]) for a, c in zip(gi, grads))
    n = _abi.cross_bwd_workspace_bytes(b, h, 1, sq, sk, d)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    out, dq = (torch.empty(b, sq, h, d, device=cuda) for _ in range(2))
    lse, dkv = torch.empty(b, h, sq, device=cuda), torch.empty(b, sk, 2, 1, d, device=cuda)
    operands = [a for t in x for a in (t.data_ptr(), t.stride()[:3])]
    shape, stream = (b, h, 1, sq, sk, d, 0.1), torch.cuda.current_stream().cuda_stream
    assert _abi.cross_fwd(*operands, lengths.data_ptr(), out.data_ptr(), lse.data_ptr(), *shape, stream) == _abi.CFA_OK
    assert _abi.cross_bwd(*operands, lengths.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                          dout.stride()[:3], dq.data_ptr(), dkv.data_ptr(), ws.data_ptr(), n, *shape,
                          stream) == _abi.CFA_OK
    cfa.check_status()
    chain = (dq.transpose(1, 2), *(dkv[:, :, i].transpose(1, 2) for i in (0, 1)))
    assert torch.equal(out.transpose(1, 2), o) and all(torch.equal(a, c) for a, c in zip(chain, grads))


def test_backward_without_room_for_its_partials(cuda):
    """2 GB of dQ partials that the allocator refuses: the least workspace, the same bits."""
    b, h, sq, sk, d = 4, 8, 4096, 8192, 64
    x = [torch.randn(b, h, s, d, device=cuda, requires_grad=True) for s in (sq, sk, sk)]
    o = cfa.cross_attention(*x, 0.125)
    dout = torch.randn_like(o)
    want = torch.autograd.grad(o, x, dout, retain_graph=True)
    size = _abi.cross_bwd_workspace_bytes_fast(b, h, h, sq, sk, d)
    assert size > 2 << 30 and _abi.cross_bwd_workspace_bytes(b, h, h, sq, sk, d) < 100 << 20
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(cuda).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + size // 2) / total)
    try:
        got = torch.autograd.grad(o, x, dout)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    cfa.check_status()

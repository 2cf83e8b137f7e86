# SPDX-License-Identifier: MIT OR Apache-2.0
"""Cross attention at the sizes and scales that tests/test_cross_gpu.py leaves out; its band."""

import math

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi
import formulas as ref
from test_cross_gpu import check, run

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


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h,hk,sq", [(2, 2, 1), (2, 2, 2), (4, 1, 2), (4, 2, 7), (2, 2, 32), (2, 2, 70)])
@pytest.mark.parametrize("scale", [0.0, -0.125, 0.3, 1.0, 4.0])
def test_scales_of_every_kernel(cuda, d, h, hk, sq, scale):
    """Scores of up to a few hundreds, zero and negative scales, for every pair of kernels.

    A score is off by delta = 44 u sum |q| |k| |scale|, u = 2^-24: two tf32 parts leave out 3 2^-22 = 12 u of a
    product, short sums of 16 truncated steps 32 u (the three-part pair: 26 u in all). P = e^(s - L) is then off
    by 2 delta (s and L), and dS = P (dP - D) by that of both its terms' absolute values, D once more by o's 2
    delta: 4 delta of the formulas with absolute values, and the sums of the products themselves (64 + n) u.
    Weights below fp32's smallest normal number, 2^-126, are zero: at scale 4 scores lie more than 87 below
    their row's largest, and what such a weight multiplies is below 2^20 here (|g| |v| d, |q| or |k|, scale)."""
    (q, k, v, dout, scale, _), _, o, grads = run(cuda, 2, h, hk, sq, 90, d, [90, 33], seed=d + sq, scale=scale)
    clean = [torch.nan_to_num(t, nan=0.0) for t in (k, v)]
    want, size = ref.cross(q, *clean, scale, [90, 33], dout)
    group = h // hk
    top = torch.matmul(q.double().abs(), clean[0].double().abs().repeat_interleave(group, 1).transpose(2, 3)).max()
    u = 2.0 ** -24
    rel = math.expm1(4 * 44 * u * float(top) * abs(scale)) + (64 + 90 + group * sq) * u
    for name, g, w, a in zip(("o", "dq", "dk", "dv"), (o, *grads), want, size):
        err = (g.detach().cpu().double() - w).abs()
        assert bool((err <= rel * a + 2.0 ** (20 - 126)).all()), f"{name}: {float((err / a.clamp_min(1e-300)).max()):.2e} of {rel:.2e}"


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 2, 5, 8, 9, 20, 32, 70])
def test_large_scores_have_weights_that_sum_to_one(cuda, d, sq):
    """The backward's weights e^(s - L), at scores near a hundred: their sum over the keys (what dV sums to for
    gradients of one) is off from the number of rows only by what L and the forward's scaled scores are rounded
    by, half a step of L each. Two uniform roundings are sqrt(2 / 3) of that in the mean square, 1.3 with what
    else there is (2^x, a quarter at this size). Scores summed in another order would be off by far more.

    One query row a head and batch element, or (from two on) rows that are copies of one another."""
    b, h, n = 40, 4, 90
    g = torch.Generator().manual_seed(d + sq)
    q = torch.randn(b, h, 1, d, generator=g).expand(b, h, sq, d)
    k, v = (torch.randn(b, h, n, d, generator=g) for _ in range(2))
    scale = 32.0 / math.sqrt(d)
    L = torch.logsumexp((q[:, :, :1].double() @ k.double().transpose(2, 3)) * scale, -1)
    x = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    o = cfa.cross_attention(*x, scale)
    dv, = torch.autograd.grad(o, x[2], torch.ones_like(o))
    total = dv[..., 0].cpu().double().sum(2) / sq
    step = 2.0 ** (torch.floor(torch.log2(L.abs())) - 24).squeeze(-1)
    off = (((total - 1.0) / step) ** 2).mean().sqrt()
    assert float(L.min()) > 16 and float(off) <= 1.3, float(off)
    cfa.check_status()


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 7, 40])
def test_a_visible_infinity_stays_in_its_batch_element(cuda, d, sq):
    """In outputs and gradients: an infinite value or key of one element leaves the others their bits."""
    g = torch.Generator().manual_seed(sq)
    x = [torch.randn(3, 2, s, d, generator=g).to(cuda) for s in (sq, 90, 90)]
    dout = torch.randn(3, 2, sq, d, generator=g).to(cuda)

    def step():
        y = [t.clone().requires_grad_(True) for t in x]
        o = cfa.cross_attention(*y, 0.125)
        return (o.detach(), *torch.autograd.grad(o, y, dout))

    want = step()
    for which in (1, 2):
        x[which][1, 0, 40, 5] = math.inf
        got = step()
        x[which][1, 0, 40, 5] = 0.0
        assert all(torch.equal(a[[0, 2]], c[[0, 2]]) for a, c in zip(got, want))
    cfa.check_status()

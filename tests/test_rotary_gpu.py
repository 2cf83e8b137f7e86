# SPDX-License-Identifier: MIT OR Apache-2.0
"""Rotary positions against the 64-bit formula (tests/formulas.py states the band), forward and
gradient, over layouts, types, sizes, strides and positions."""

import math

import pytest
import torch

import candle_fused_attn as cfa
import formulas as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(got, want, band):
    err = (got.detach().cpu().double() - want).abs()
    assert bool((err <= band).all()), f"off by up to {(err - band).max():.2e} beyond the band"


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,s,d,rot", [
    (1, 1, 1, 2, 2), (2, 3, 5, 64, 64), (1, 6, 240, 64, 64), (3, 2, 17, 128, 64), (2, 5, 9, 40, 40),
    (1, 4, 33, 80, 20), (2, 1, 7, 33, 30), (1, 2, 3, 32, 0), (2, 40, 11, 128, 128),
    (1, 3, 700, 256, 2), (1, 70, 2, 1024, 1024), (5, 1, 1, 96, 94)])
def test_forward_and_gradient(cuda, dtype, interleaved, b, h, s, d, rot):
    g = torch.Generator().manual_seed(b * 1000 + s + d)
    x = torch.randn(b, h, s, d, generator=g).to(dtype).to(cuda).requires_grad_(True)
    dy = torch.randn(b, h, s, d, generator=g).to(dtype).to(cuda)
    pos = torch.randint(0, 5000, (b, s), generator=g).to(cuda)
    freqs = 10000.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64, device=cuda) / max(rot, 1))
    y = cfa.rotary(x, pos, freqs, amplitude=1.25, interleaved=interleaved)
    assert y.shape == x.shape and y.dtype == dtype and y.transpose(1, 2).is_contiguous()
    check(y, ref.rotate(x, pos, freqs, 1.25, interleaved),
          ref.rotate_band(x, freqs, 1.25, interleaved, dtype))
    (dx,) = torch.autograd.grad(y, x, dy)
    check(dx, ref.rotate(dy, pos, freqs, 1.25, interleaved, inverse=True),
          ref.rotate_band(dy, freqs, 1.25, interleaved, dtype))
    cfa.check_status()


@pytest.mark.parametrize("start", [0, 100_000, 2 ** 24 + 1, 2 ** 31 - 200, 2 ** 40])
def test_far_positions_keep_their_angles(cuda, start):
    """fp32 products would be off by whole radians here; the band does not grow with the position
    (the 64-bit product's own rounding is start 2^-53 radians)."""
    x = torch.randn(1, 2, 100, 64, generator=torch.Generator().manual_seed(3)).to(cuda)
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    pos = torch.arange(start, start + 100, device=cuda)
    want = ref.rotate(x, pos, freqs)
    band = ref.rotate_band(x, freqs) + 4 * start * 2.0 ** -53 * x.cpu().abs().amax().item()
    check(cfa.rotary(x, pos, freqs), want, band)
    check(cfa.rotary(x, start, freqs), want, band)  # an int: consecutive positions
    if start + 100 < 2 ** 31:
        check(cfa.rotary(x, pos.int(), freqs), want, band)


def test_position_shapes_and_negative_positions(cuda):
    x = torch.randn(3, 2, 4, 32, generator=torch.Generator().manual_seed(4)).to(cuda)
    freqs, _ = cfa.rotary_frequencies(32, device=cuda)
    p = torch.tensor([-5, 0, 7, 1000], device=cuda)
    want, band = ref.rotate(x, p, freqs), ref.rotate_band(x, freqs)
    for pos in (p, p[None], p.expand(3, 4), p.repeat(2)[:8:1][:4], torch.stack([p, p], 1)[:, 0]):
        check(cfa.rotary(x, pos, freqs), want, band)
    each = torch.tensor([[3], [9], [27]], device=cuda)
    check(cfa.rotary(x, each, freqs), ref.rotate(x, each, freqs), band)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides_and_alignment(cuda, dtype, interleaved):
    """Views of a projection, rows at odd offsets, transposed and expanded inputs: the same values."""
    g = torch.Generator().manual_seed(8)
    base = torch.randn(2, 9, 3, 4, 72, generator=g).to(dtype).to(cuda)
    freqs, _ = cfa.rotary_frequencies(32, device=cuda)
    wide = torch.randn(2, 4, 64, 9, generator=g).to(dtype).to(cuda)
    one = torch.randn(1, 1, 9, 64, generator=g).to(dtype).to(cuda)
    for x in (base[:, :, 1, :, :64].transpose(1, 2), base[:, :, 0, :, 1:65].transpose(1, 2),
              base[:, :, 2, :, 2:66].transpose(1, 2), base[:, ::2, 1, ::3, 8:].transpose(1, 2),
              wide.transpose(2, 3), one.expand(2, 4, 9, 64)):
        y = cfa.rotary(x, 11, freqs, interleaved=interleaved)
        pos = torch.arange(11, 11 + x.shape[2])
        check(y, ref.rotate(x, pos, freqs, 1.0, interleaved),
              ref.rotate_band(x, freqs, 1.0, interleaved, dtype))
    # an expanded leaf: the gradient sums over what shares it
    leaf = one.float().requires_grad_(True)
    dy = torch.randn(2, 4, 9, 64, generator=g).to(cuda)
    cfa.rotary(leaf.expand(2, 4, 9, 64), 11, freqs, interleaved=interleaved).backward(dy)
    each = ref.rotate(dy, torch.arange(11, 20), freqs, 1.0, interleaved, inverse=True)
    band = ref.rotate_band(dy, freqs, 1.0, interleaved).sum((0, 1), keepdim=True)
    want = each.sum((0, 1), keepdim=True)
    # eight addends, seven roundings of at most the partial sums
    check(leaf.grad, want, band + 7 * 2.0 ** -24 * each.abs().sum((0, 1), keepdim=True))


def test_qkv_rotates_queries_and_keys_only(cuda):
    b, s, h, d = 2, 37, 3, 64
    qkv = torch.randn(b, s, 3 * h * d, generator=torch.Generator().manual_seed(5)).to(cuda)
    freqs, amp = cfa.rotary_frequencies(d, scaling="yarn", factor=4.0, original_length=1024,
                                        device=cuda)
    x = qkv.clone().requires_grad_(True)
    y = cfa.rotary_qkv(x, h, 50, freqs, amplitude=amp)
    got, src = y.view(b, s, 3, h, d), qkv.view(b, s, 3, h, d)
    pos = torch.arange(50, 50 + s)
    for i in range(2):
        part = src[:, :, i].transpose(1, 2)
        check(got[:, :, i].transpose(1, 2), ref.rotate(part, pos, freqs, amp),
              ref.rotate_band(part, freqs, amp))
    assert torch.equal(got[:, :, 2], src[:, :, 2])
    dy = torch.randn(b, s, 3 * h * d, generator=torch.Generator().manual_seed(6)).to(cuda)
    y.backward(dy)
    g, dsrc = x.grad.view(b, s, 3, h, d), dy.view(b, s, 3, h, d)
    for i in range(2):
        part = dsrc[:, :, i].transpose(1, 2)
        check(g[:, :, i].transpose(1, 2), ref.rotate(part, pos, freqs, amp, inverse=True),
              ref.rotate_band(part, freqs, amp))
    assert torch.equal(g[:, :, 2], dsrc[:, :, 2])
    # a strided projection and 16-bit types read in place
    wide = torch.randn(b, s, 3 * h * d + 5, device=cuda).to(BF16)[..., 3:3 * h * d + 3]
    got = cfa.rotary_qkv(wide, h, 0, freqs, interleaved=True)
    assert torch.equal(got, cfa.rotary_qkv(wide.contiguous(), h, 0, freqs, interleaved=True))


def test_gradient_against_differences(cuda):
    """The operator is linear in x, so a central difference is exact up to fp32's roundings: the two
    outputs are off by 9 steps each of values up to 6, over 2 eps."""
    g = torch.Generator().manual_seed(7)
    x, u, w = (torch.randn(1, 2, 6, 16, generator=g).to(cuda) for _ in range(3))
    freqs, _ = cfa.rotary_frequencies(12, device=cuda)
    leaf = x.clone().requires_grad_(True)
    (cfa.rotary(leaf, 3, freqs) * w).sum().backward()
    eps = 0.5
    hi, lo = (cfa.rotary(x + sgn * eps * u, 3, freqs).double() for sgn in (1, -1))
    diff = ((hi - lo) * w.double()).sum().item() / (2 * eps)
    band = 2 * 10 * 2.0 ** -24 * 6 * w.abs().sum().item() / (2 * eps)
    assert abs(diff - (leaf.grad.double() * u.double()).sum().item()) <= band


def test_empty(cuda):
    freqs, _ = cfa.rotary_frequencies(32, device=cuda)
    for shape in ((0, 2, 3, 32), (2, 0, 3, 32), (2, 3, 0, 32)):
        x = torch.empty(shape, device=cuda, requires_grad=True)
        y = cfa.rotary(x, 0, freqs)
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape
    cfa.check_status()


def test_non_finite_values_stay_in_their_pairs(cuda):
    x = torch.ones(1, 1, 2, 8, device=cuda)
    x[0, 0, 0, 1] = math.inf
    x[0, 0, 1, 7] = math.nan
    freqs, _ = cfa.rotary_frequencies(4, device=cuda)
    y = cfa.rotary(x, 1, freqs)
    assert not y[0, 0, 0, [1, 3]].isfinite().any()
    assert y[0, 0, 0, [0, 2, 4, 5, 6, 7]].isfinite().all()
    assert y[0, 0, 1, 7].isnan() and y[0, 0, 1, :7].isfinite().all()


def test_other_stream_and_graph(cuda):
    x = torch.randn(2, 3, 40, 64, device=cuda)
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    pos = torch.arange(40, device=cuda)
    want = cfa.rotary(x, pos, freqs)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = cfa.rotary(x, pos, freqs)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cfa.rotary(x, pos, freqs)
    pos += 5
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, cfa.rotary(x, pos, freqs)) and not torch.equal(out, want)


def test_second_derivative_is_refused(cuda):
    """Not dropped: an error where the gradient itself is differentiated, none where it only could be."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    x = torch.randn(1, 2, 5, 64, device=cuda, requires_grad=True)
    for y in (cfa.rotary(x, 3, freqs), cfa.cross_attention(x, x, x, 0.125)):
        dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True, retain_graph=True)
        want, = torch.autograd.grad((y * y).sum(), x)
        assert torch.equal(dx, want)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            dx.sum().backward()

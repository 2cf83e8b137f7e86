# SPDX-License-Identifier: MIT OR Apache-2.0
"""What paged_attention keeps of the softmax's weights: scores that are exact (one dim of q and k is not
zero, the scale is one), so that only the weights' own precision shows."""

import math

import pytest
import torch

import candle_fused_attn as cfa
import formulas as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def attend(cuda, scores, v, h, d, qt, kt):
    """scores [b, n] (of the cache's type) and v [b, n, d] -> o [b, h, d] (float64): every head's query is
    the first unit vector."""
    b, n = scores.shape
    k = torch.zeros(b, 1, n, d, dtype=kt)
    k[:, 0, :, 0] = scores.to(kt)
    q = torch.zeros(b, h, 1, d, dtype=qt)
    q[..., 0] = 1.0
    gen = torch.Generator().manual_seed(1)
    kc, vc, table, lengths = ref.paged(list(k), list(v[:, None].to(kt)), 16, gen, kt)
    o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), 1.0)
    cfa.check_status()
    return o[:, :, 0].cpu().double()


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h", [1, 4, 8])
def test_bf16_outputs_have_weights_of_24_bits(cuda, d, h):
    """Two keys whose weighted values nearly cancel, v = 1 and -c with c the bf16 number next to e^t: the
    result (1 - e^-t c) / (1 + e^-t) is below 2^-8, and its own bf16 step hides no more than 2^-8 of that.
    The weight e^-t, t < 1.5, is off by 6 u (the exponent's argument, below 2.2, rounds once and its
    constant is off by a quarter step: 1.9 u; 2^x: 4 u), the parts and the truncated sums of two terms of 1
    add 3 u, the quotient 2 u of the result: 12 u / (1 + e^-t) in all. Weights of 16 bits are 64 u off."""
    b = 512
    g = torch.Generator().manual_seed(d + h)
    t = (0.5 + torch.rand(b, generator=g)).bfloat16().double()
    c = t.exp().bfloat16().double()
    v = torch.stack((torch.ones(b, dtype=torch.float64), -c), 1)[:, :, None].expand(b, 2, d)
    scores = torch.stack((torch.zeros(b, dtype=torch.float64), -t), 1)
    o = attend(cuda, scores, v, h, d, BF16, BF16)
    p = torch.exp(-t)
    want = ((1.0 - p * c) / (1.0 + p))[:, None, None]
    lim = torch.finfo(BF16).eps / 2 * want.abs() + 12 * U / (1.0 + p)[:, None, None]
    assert bool(((o - want).abs() <= lim).all()), float(((o - want).abs() / lim).max())


@pytest.mark.parametrize("qt", [F32, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h", [2, 24])
def test_a_tail_of_small_weights_over_fp16_counts(cuda, qt, d, h):
    """One key takes nearly all of the weight and has the value 0; 600 others of e^-16 to e^-8 share values
    near 1. A weight is off by 24 u (the argument, below 23, rounds once and its constant is off by a
    quarter step: 20 u; 2^x: 4 u), its two parts by 2^-22 = 4 u of it and 2^-39; the sums of n terms in
    chunks by (n / 16 + 64) u; l by 24 u."""
    b, n = 4, 601
    g = torch.Generator().manual_seed(d + h)
    scores = (-16.0 + 8.0 * torch.rand(b, n, generator=g)).half().double()
    v = (0.5 + torch.rand(b, n, d, generator=g)).half().double()
    scores[:, 100], v[:, 100] = 0.0, 0.0
    o = attend(cuda, scores, v, h, d, qt, F16)
    want = torch.softmax(scores, 1)[:, None] @ v
    lim = (24 + 4 + n / 16 + 64 + 24) * U * want + 2.0 ** -39 * v.sum(1, keepdim=True)
    if qt == F16:
        lim = lim + torch.finfo(F16).eps / 2 * want + 2.0 ** -25
    assert bool(((o - want).abs() <= lim).all()), float(((o - want).abs() / lim).max())


@pytest.mark.parametrize("qt,kt", [(F32, F32), (F32, BF16), (F32, F16), (F16, F16), (BF16, BF16)])
@pytest.mark.parametrize("h", [1, 2, 8, 24])
def test_a_visible_infinity_stays_in_its_sequence(cuda, qt, kt, h):
    """An infinite value: its dim of that sequence is not finite, everything else as without it. An infinite
    key (scores of both signs: a weight of zero, or none that is defined): the other sequences as without it."""
    g = torch.Generator().manual_seed(h)
    k, v = ([torch.randn(1, n, 64, generator=g).to(kt) for n in (100, 100, 700)] for _ in range(2))
    q = torch.randn(3, h, 1, 64, generator=g).to(qt).to(cuda)

    def attend():
        kc, vc, table, lengths = (t.to(cuda) for t in ref.paged(k, v, 16, torch.Generator().manual_seed(1), kt))
        return cfa.paged_attention(q, kc, vc, table, lengths, 0.125)

    want = attend()
    v[1][0, 40, 7] = math.inf
    got = attend()
    assert not got[1, :, 0, 7].isfinite().any()
    got[1, :, 0, 7] = want[1, :, 0, 7]
    assert torch.equal(got, want)
    v[1][0, 40, 7] = 0.0
    k[1][0, 40, 7] = math.inf
    assert torch.equal(attend()[[0, 2]], want[[0, 2]])
    cfa.check_status()

# SPDX-License-Identifier: MIT OR Apache-2.0
"""What autograd sees of the operators on the GPU: second derivatives, in-place writes."""

import pytest
import torch

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sq", [3, 70])
@pytest.mark.parametrize("by", ["q", "k", "v"])
@pytest.mark.parametrize("loss", ["sum", "weighted"])
def test_second_derivatives_of_cross_attention_are_refused(cuda, sq, by, loss):
    """The gradients depend on q, k and v as well as on the incoming gradient: one that is constant (o.sum())
    does not make them constants. A gradient penalty would lose its terms without a word."""
    x = {n: torch.randn(2, 2, s, 64, device=cuda) for n, s in (("q", sq), ("k", 90), ("v", 90))}
    x[by].requires_grad_(True)
    o = cfa.cross_attention(x["q"], x["k"], x["v"], 0.125)
    upstream = o.sum() if loss == "sum" else (o * torch.randn_like(o)).sum()
    g, = torch.autograd.grad(upstream, x[by], create_graph=True)
    other = x[by].square().sum()
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        g.square().sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        (g.square().sum() + other).backward()


def test_a_rotation_of_a_constant_gradient_is_constant(cuda):
    """dx = R^T dy holds no x: nothing of it is differentiable, and nothing is lost."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    x = torch.randn(1, 2, 8, 64, device=cuda, requires_grad=True)
    g, = torch.autograd.grad(cfa.rotary(x, 3, freqs).sum(), x, create_graph=True)
    assert not g.requires_grad
    (g.square().sum() + x.square().sum()).backward()
    assert torch.equal(x.grad, 2 * x)

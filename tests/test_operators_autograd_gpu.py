# SPDX-License-Identifier: MIT OR Apache-2.0
"""What autograd sees of the operators on the GPU: second derivatives, in-place writes."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi

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


@pytest.mark.parametrize("which", ["k", "v"])
def test_append_is_seen_as_an_in_place_write(cuda, which):
    """A backward that saved the cache (or a view of it) before new tokens were written raises, as after any
    in-place operation."""
    pool = torch.randn(2, 3, 16, 2, 64, device=cuda)
    caches = dict(k=pool[0], v=pool[1].clone())
    w = torch.ones(64, device=cuda, requires_grad=True)
    x = torch.randn(1, 2, 1, 64, device=cuda)
    table, lengths = (torch.ones(1, n, dtype=torch.int32, device=cuda) for n in (3, 1))

    def append():
        cfa.paged_append(x, x, caches["k"], caches["v"], table, lengths.view(-1))

    append()
    y = (caches[which][1:] * w).sum()
    y.backward(retain_graph=True)
    with torch.no_grad():
        append()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    cfa.check_status()


def test_append_into_inference_tensors(cuda):
    """They have no version to count."""
    with torch.inference_mode():
        k, v = torch.zeros(2, 3, 16, 2, 64, device=cuda).unbind(0)
        x = torch.randn(1, 2, 1, 64, device=cuda)
        table, lengths = torch.ones(1, 3, dtype=torch.int32, device=cuda), torch.ones(1, dtype=torch.int32, device=cuda)
        cfa.paged_append(x, x, k, v, table, lengths)
    cfa.paged_append(x, x, k, v, table, lengths)
    assert torch.equal(k[1, 0], x[0, :, 0]) and torch.equal(v[1, 0], x[0, :, 0])
    cfa.check_status()


@pytest.mark.parametrize("op", ["cross", "rotary"])
def test_a_failed_capture_is_an_error(cuda, op):
    """A backward captured while an eager graph of the same leaf lives: torch synchronises with the stream of
    that graph's gradient node, which ends the capture (plain operations fare alike). It has to come out as an
    error, and calls have to go on."""
    package = Path(__file__).resolve().parents[1] / "candle-fused-attn_b200"
    code = f"""
import sys, warnings; sys.path.insert(0, {str(package)!r}); warnings.simplefilter("ignore")
import torch, candle_fused_attn as cfa
freqs, _ = cfa.rotary_frequencies(64)
k = torch.randn(1, 2, 90, 64, device="cuda")
op = dict(cross=lambda x: cfa.cross_attention(x, k, k, 0.1), rotary=lambda x: cfa.rotary(x, 3, freqs))[{op!r}]
x = torch.randn(1, 2, 40, 64, device="cuda", requires_grad=True)
want, = torch.autograd.grad(op(x).square().sum(), x)
eager = op(x)
try:
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        op(x).square().sum().backward()
except RuntimeError as e:
    print("refused")
eager.square().sum().backward()
x.grad = None
op(x).square().sum().backward()
cfa.check_status()
print("same" if torch.equal(x.grad, want) else "other")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("same\n"), r.stdout + r.stderr


@pytest.mark.parametrize("op", ["cross", "rotary"])
def test_an_error_in_a_backward_is_raised(cuda, op):
    """A bounded wait of an earlier kernel expires between forward and backward: the backward, in autograd's own
    thread, raises what a call does, and the next one runs."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    x = torch.randn(1, 2, 40, 64, device=cuda, requires_grad=True)
    o = cfa.cross_attention(x, x, x, 0.1) if op == "cross" else cfa.rotary(x, 3, freqs)
    want, = torch.autograd.grad(o.square().sum(), x, retain_graph=True)
    ws = torch.zeros(256, dtype=torch.uint8, device=cuda)
    stream = torch.cuda.current_stream().cuda_stream
    assert _abi.selftest_bounded_wait(ws.data_ptr(), 20_000_000, 2, stream) == _abi.CFA_OK
    torch.cuda.synchronize()
    with pytest.raises(cfa.FusedAttentionError, match="expired"):
        torch.autograd.grad(o.square().sum(), x, retain_graph=True)
    got, = torch.autograd.grad(o.square().sum(), x)
    assert torch.equal(got, want)
    cfa.check_status()


def test_function_transforms_are_refused(cuda):
    """Tensors of torch.func have no memory of their own: an error, not a wrong result."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    x = torch.randn(2, 1, 2, 9, 64, device=cuda)
    for call in (lambda t: cfa.cross_attention(t, t, t, 0.1), lambda t: cfa.rotary(t, 3, freqs)):
        for run in (lambda: torch.vmap(call)(x), lambda: torch.func.grad(lambda t: call(t).sum())(x[0]),
                    lambda: torch.func.jvp(call, (x[0],), (x[0],))):
            with pytest.raises(RuntimeError):
                run()

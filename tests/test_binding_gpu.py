# SPDX-License-Identifier: MIT OR Apache-2.0
"""The operators' compiled Python side: what autograd, devices, threads and odd operands ask of it."""

import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import candle_fused_attn as cfa

pytestmark = pytest.mark.gpu


def offset(shape, cuda, by=1):
    """A dense tensor whose rows start `by` elements off 16 bytes."""
    n = 1
    for x in shape:
        n *= x
    return torch.randn(n + by, device=cuda)[by:].view(shape)


@pytest.mark.parametrize("grad", [False, True])
def test_dense_operands_off_16_bytes_are_copied(cuda, grad):
    q, k, v = (offset((2, 2, s, 64), cuda) for s in (40, 70, 70))
    copies = [t.clone() for t in (q, k, v)]
    for t in (q, k, v, *copies):
        t.requires_grad_(grad)
    got, want = cfa.cross_attention(q, k, v, 0.125), cfa.cross_attention(*copies, 0.125)
    assert torch.equal(got, want)
    if grad:
        dout = offset((2, 2, 40, 64), cuda, 3)
        a = torch.autograd.grad(got, (q, k, v), dout)
        b = torch.autograd.grad(want, copies, dout.clone())
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_one_head_with_an_odd_stride(cuda):
    """A dimension of one may have any stride."""
    k = torch.randn(2, 70, 64, device=cuda).as_strided((2, 1, 70, 64), (70 * 64, 7, 64, 1))
    q = torch.randn(2, 3, 5, 64, device=cuda)
    want = cfa.cross_attention(q, k.clone(memory_format=torch.contiguous_format), k.contiguous(), 0.125)
    assert torch.equal(cfa.cross_attention(q, k, k, 0.125), want)


def test_saved_tensors_are_watched(cuda):
    """Positions, keys or outputs changed between forward and backward are an error, not a wrong gradient."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    x = torch.randn(1, 2, 8, 64, device=cuda, requires_grad=True)
    at = torch.arange(8, device=cuda)
    y = cfa.rotary(x, at, freqs)
    at += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    k = torch.randn(1, 2, 8, 64, device=cuda)
    o = cfa.cross_attention(x, k, k, 0.125)
    k.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    o = cfa.cross_attention(x, x, x, 0.125)
    with torch.no_grad():
        o.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()


def test_checkpointing_recomputes_the_same(cuda):
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    k = torch.randn(2, 1, 30, 64, device=cuda)

    def layer(x):
        return cfa.cross_attention(cfa.rotary(x, 5, freqs), k, k, 0.125)

    grads = []
    for run in (layer, lambda x: checkpoint(layer, x, use_reentrant=False)):
        x = torch.nn.Parameter(torch.linspace(-1, 1, 2 * 4 * 9 * 64, device=cuda).view(2, 4, 9, 64))
        (run(x) ** 2).sum().backward()
        grads.append(x.grad)
    assert torch.equal(*grads)


def test_gradients_of_some_inputs_only(cuda):
    q, k = torch.randn(1, 2, 33, 64, device=cuda), torch.randn(1, 2, 50, 64, device=cuda)
    full = [t.clone().requires_grad_(True) for t in (q, k, k)]
    want = torch.autograd.grad(cfa.cross_attention(*full, 0.125).square().sum(), full)
    for i in range(3):
        x = [t.clone() for t in (q, k, k)]
        x[i].requires_grad_(True)
        g, = torch.autograd.grad(cfa.cross_attention(*x, 0.125).square().sum(), x[i])
        assert torch.equal(g, want[i])
    shared = k.clone().requires_grad_(True)  # one tensor as both: its gradients are added
    g, = torch.autograd.grad(cfa.cross_attention(q, shared, shared, 0.125).square().sum(), shared)
    assert torch.equal(g, want[1] + want[2])


def test_threads_call_at_once(cuda):
    """Four threads on streams of their own, forward and backward: each its own results."""
    freqs, _ = cfa.rotary_frequencies(64, device=cuda)
    inputs = [torch.randn(2, 4, 100 + i, 64, device=cuda) for i in range(4)]
    torch.cuda.synchronize()

    def work(x):
        x = x.clone().requires_grad_(True)
        y = cfa.cross_attention(cfa.rotary(x, 3, freqs), x, x, 0.125)
        return y.detach(), *torch.autograd.grad(y.square().sum(), x)

    want = [work(x) for x in inputs]
    torch.cuda.synchronize()
    got = [None] * 4

    def loop(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = work(inputs[i])
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_operands_of_another_device_are_refused(cuda):
    q, k = torch.zeros(1, 2, 3, 64, device=cuda), torch.zeros(1, 2, 5, 64, device=cuda)
    for call in (lambda: cfa.cross_attention(q, k.cpu(), k, 0.125),
                 lambda: cfa.cross_attention(q, k, k, 0.125, torch.ones(1, dtype=torch.int32)),
                 lambda: cfa.rotary(q, 0, torch.ones(4, dtype=torch.float64)),
                 lambda: cfa.rotary(q, torch.arange(3), torch.ones(4, dtype=torch.float64, device=cuda))):
        with pytest.raises(cfa.FusedAttentionError, match="CUDA tensors required"):
            call()

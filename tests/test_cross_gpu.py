# SPDX-License-Identifier: MIT OR Apache-2.0
"""Cross attention, forward and gradients, against the 64-bit formula (tests/formulas.py).

The band is the fused attention's, 1e-5 relative, normwise, here of every (batch, head) slice: it
follows from the split products' error model (tests/test_linear_gpu.py), by which scores are off by
26 2^-24 sum |q| |k| scale, 8e-6 at d = 64 and unit inputs, p by that factor and 2^-22, both averaged
down in the sums. (d = 128: two tf32 parts an operand leave out at most 3 2^-22 |q| |k| of a product.) To it come 26 2^-24 of the same sums over absolute values: dP - D cancels (for a
single key to nothing), and what dP and D are off by stays.
"""

import math

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi
import formulas as ref

pytestmark = pytest.mark.gpu

BAND = 1e-5


def make(b, h, hk, sq, sk, d, lens, seed=0, fill=float("nan")):
    """q, k, v, dout (CPU), k and v holding `fill` behind the lengths."""
    g = torch.Generator().manual_seed(seed)
    q, dout = (torch.randn(b, sq, h, d, generator=g).transpose(1, 2) for _ in range(2))
    kv = torch.randn(b, sk, 2, hk, d, generator=g)
    if lens is not None:
        for i, n in enumerate(lens):
            kv[i, max(0, n):] = fill
    return q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2), dout


def near(got, want, size, name):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, name
    norm = lambda t: t.flatten(2).norm(dim=2)  # noqa: E731
    off = norm(got - want) - BAND * norm(want) - 26 * 2.0 ** -24 * norm(size)
    assert bool((off <= 0).all()), f"{name}: {float((norm(got - want) / norm(want)).max()):.2e}"


def run(cuda, b, h, hk, sq, sk, d, lens, seed=0, scale=None):
    q, k, v, dout = make(b, h, hk, sq, sk, d, lens, seed)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    lengths = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=cuda)
    x = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
    o = cfa.cross_attention(*x, scale, key_lengths=lengths)
    grads = torch.autograd.grad(o, x, dout.to(cuda))
    cfa.check_status()
    return (q, k, v, dout, scale, lengths), x, o, grads


def check(cuda, b, h, hk, sq, sk, d, lens, seed=0, scale=None):
    (q, k, v, dout, scale, lengths), x, o, grads = run(cuda, b, h, hk, sq, sk, d, lens, seed, scale)
    clean = [torch.nan_to_num(t, nan=0.0) for t in (k, v)]
    want, size = ref.cross(q, *clean, scale, lens, dout)
    assert o.transpose(1, 2).is_contiguous()
    for name, g, w, a in zip(("o", "dq", "dk", "dv"), (o, *grads), want, size):
        near(g, w, a, name)
    if lens is not None:
        for i, n in enumerate(lens):
            n = max(0, n)
            assert not grads[1][i, :, n:].any() and not grads[2][i, :, n:].any()
            if n == 0:
                assert not o[i].any() and not grads[0][i].any()
    with torch.no_grad():  # the forward of its own: few rows split over the keys, or the same kernel
        near(cfa.cross_attention(*x, scale, key_lengths=lengths), want[0], size[0], "o without gradients")
    cfa.check_status()


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b,h,hk,sq,sk", [
    (1, 1, 1, 1, 1), (2, 3, 3, 7, 5), (1, 2, 2, 1, 300), (2, 2, 1, 64, 128), (1, 6, 2, 65, 129),
    (3, 4, 4, 257, 100), (2, 8, 1, 33, 63), (1, 4, 2, 300, 700), (1, 2, 2, 513, 1), (1, 9, 3, 5, 1000)])
def test_shapes(cuda, d, b, h, hk, sq, sk):
    check(cuda, b, h, hk, sq, sk, d, None, seed=sq + sk)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h,hk,sq,sk,lens", [
    (2, 2, 40, 70, [70, 0, 1, 69]), (4, 2, 130, 300, [128, 129, 300, 0]), (3, 1, 1, 200, [0, 200, 64, 65]),
    (2, 1, 20, 130, [-3, 1000, 0, 130]), (2, 2, 300, 64, [0, 0, 0, 0])])
def test_key_lengths(cuda, d, h, hk, sq, sk, lens):
    """Padded batches, the padding holding NaN; lengths are held within 0 .. sk."""
    check(cuda, len(lens), h, hk, sq, sk, d, [max(0, min(sk, n)) for n in lens], seed=sk)
    q, k, v, _ = make(len(lens), h, hk, sq, sk, d, [max(0, min(sk, n)) for n in lens])
    args = [t.to(cuda) for t in (q, k, v)]
    a, c = (cfa.cross_attention(*args, 0.1, key_lengths=torch.tensor(x, dtype=torch.int32, device=cuda))
            for x in (lens, [max(0, min(sk, n)) for n in lens]))
    assert torch.equal(a, c)


@pytest.mark.parametrize("d,sq,sk,h,hk", [(64, 100, 2500, 4, 2), (32, 70, 2100, 2, 1), (128, 80, 1100, 4, 2),
                                          (64, 513, 2048, 2, 2), (128, 65, 1024, 2, 1)])
def test_long_key_sequences(cuda, d, sq, sk, h, hk):
    """Many key blocks: their dQ partials summed by the last of them, or by a kernel of its own."""
    check(cuda, 2, h, hk, sq, sk, d, [sk, sk // 2 + 3], seed=d)


@pytest.mark.parametrize("d,h,hk,sq,sk", [(64, 8, 4, 300, 900), (32, 3, 1, 130, 700), (128, 4, 2, 200, 400),
                                          (64, 1, 1, 1500, 150)])
def test_turn_chain_gives_the_same_bits(cuda, d, h, hk, sq, sk):
    """The workspace too small for the dQ partials (what more than 4 GB of them are): key blocks add to
    dQ in turn, the same sums in the same order."""
    b, lens = 3, [sk, sk // 2, 0]
    (_, _, _, dout, scale, lengths), x, o, grads = run(cuda, b, h, hk, sq, sk, d, lens)
    q, k, v = (t.detach() for t in x)
    dout = dout.to(cuda)
    n = _abi.cross_bwd_workspace_bytes(b, h, hk, sq, sk, d)
    assert n < _abi.cross_bwd_workspace_bytes_fast(b, h, hk, sq, sk, d)
    ws = torch.empty(n, dtype=torch.uint8, device=cuda)
    o2, dq = (torch.empty(b, sq, h, d, device=cuda) for _ in range(2))
    lse, dkv = torch.empty(b, h, sq, device=cuda), torch.empty(b, sk, 2, hk, d, device=cuda)
    operands = [a for t in (q, k, v) for a in (t.data_ptr(), t.stride()[:3])]
    shape, stream = (b, h, hk, sq, sk, d, scale), torch.cuda.current_stream().cuda_stream
    assert _abi.cross_fwd(*operands, lengths.data_ptr(), o2.data_ptr(), lse.data_ptr(), *shape,
                          stream) == _abi.CFA_OK
    assert _abi.cross_bwd(*operands, lengths.data_ptr(), o2.data_ptr(), lse.data_ptr(), dout.data_ptr(),
                          dout.stride()[:3], dq.data_ptr(), dkv.data_ptr(), ws.data_ptr(), n, *shape,
                          stream) == _abi.CFA_OK
    cfa.check_status()
    chain = (dq.transpose(1, 2), *(dkv[:, :, i].transpose(1, 2) for i in (0, 1)))
    assert torch.equal(o, o2.transpose(1, 2)) and all(torch.equal(y, z) for y, z in zip(grads, chain))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h,hk,sq", [(2, 2, 1), (8, 1, 1), (3, 1, 3), (4, 2, 8), (17, 1, 1), (2, 2, 32), (3, 1, 11)])
def test_few_query_rows(cuda, d, h, hk, sq):
    """1, 8, 9, 16, 17, 32 and 33 query rows a key head: the kernels of few rows, and one row over; lengths
    that end in the first and the last of a block's tiles, on a block's end, one key, none."""
    check(cuda, 6, h, hk, sq, 300, d, [300, 128, 17, 1, 0, 129], seed=sq + h)
    check(cuda, 1, h, hk, sq, 64, d, None, seed=sq)
    check(cuda, 2, h, hk, sq, 1030, d, [1030, 700], seed=h)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("b,h,hk,sq,sk,lens", [
    (1, 8, 1, 500, 200, None), (1, 1, 1, 1000, 130, [90]), (2, 6, 1, 700, 300, [300, 0]),
    (3, 16, 2, 200, 1000, [1000, 64, 129]), (1, 2, 1, 2000, 2300, [2300]), (2, 4, 1, 1100, 64, [64, 1])])
def test_few_key_blocks(cuda, d, b, h, hk, sq, sk, lens):
    """Few key blocks a batch element: a key block's query tiles run in parts on several SMs, their dK,
    dV summed in order by a kernel of its own, and dQ's partials too (or by the turn chain)."""
    check(cuda, b, h, hk, sq, sk, d, lens, seed=sq)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 3, 10, 31, 63, 65])
def test_short_groups_share_tiles(cuda, d, sq):
    """The query rows of a group lie behind one another in the tiles: heads that begin inside one."""
    check(cuda, 2, 15, 3, sq, 150, d, [150, 77], seed=sq)


@pytest.mark.parametrize("d", [32, 64, 128])
def test_bitwise_reruns_and_batches(cuda, d):
    """Reruns, and a batch element alone, give the same bits in every output."""
    lens = [130, 20, 300]
    (q, k, v, dout, scale, lengths), _, o, grads = run(cuda, 3, 4, 2, 150, 300, d, lens)
    again = run(cuda, 3, 4, 2, 150, 300, d, lens)
    assert torch.equal(o, again[2]) and all(torch.equal(a, c) for a, c in zip(grads, again[3]))
    for i in range(3):
        x = [t[i:i + 1].to(cuda).requires_grad_(True) for t in (q, k, v)]
        oi = cfa.cross_attention(*x, scale, key_lengths=lengths[i:i + 1])
        gi = torch.autograd.grad(oi, x, dout[i:i + 1].to(cuda))
        assert torch.equal(oi[0], o[i]) and all(torch.equal(a[0], c[i]) for a, c in zip(gi, grads))


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sq", [1, 7, 30])
def test_few_rows_do_not_depend_on_the_batch(cuda, d, sq):
    """Outputs and gradients of each batch element alone, bit for bit."""
    lens = [900, 1, 0, 257, 64]
    (q, k, v, dout, scale, lengths), _, o, grads = run(cuda, 5, 4, 4, sq, 900, d, lens, scale=0.1)
    for i in range(5):
        x = [t[i:i + 1].to(cuda).requires_grad_(True) for t in (q, k, v)]
        o1 = cfa.cross_attention(*x, scale, key_lengths=lengths[i:i + 1])
        g1 = torch.autograd.grad(o1, x, dout[i:i + 1].to(cuda))
        assert torch.equal(o1[0], o[i]) and all(torch.equal(a[0], b[i]) for a, b in zip(g1, grads))


def test_equal_lengths_match_the_fused_attention(cuda):
    """Keys as long as the queries, a head each: fused_attention's own result, bit for bit (at 128 the two
    run on different units)."""
    for d in (32, 64):
        q, k, v, dout = make(2, 3, 3, 200, 200, d, None)
        res = []
        for fn in (lambda *x: cfa.cross_attention(*x, 0.2), lambda *x: cfa.fused_attention(*x, 0.2, False)):
            x = [t.to(cuda).requires_grad_(True) for t in (q, k, v)]
            o = fn(*x)
            res.append((o, *torch.autograd.grad(o, x, dout.to(cuda))))
        assert all(torch.equal(a, c) for a, c in zip(*res))


def test_strides_alignment_and_shared_inputs(cuda):
    b, h, sq, sk, d = 2, 4, 30, 50, 64
    q, k, v, dout = (t.to(cuda) for t in make(b, h, h, sq, sk, d, None))
    want = cfa.cross_attention(q, k, v, 0.125)
    odd = torch.zeros(b, h, sk, d + 1, device=cuda)
    odd[..., 1:] = k
    assert torch.equal(cfa.cross_attention(q.contiguous(), odd[..., 1:], v.contiguous(), 0.125), want)
    wide = v.transpose(2, 3).contiguous().transpose(2, 3)  # d not contiguous
    assert torch.equal(cfa.cross_attention(q, k, wide, 0.125), want)
    # one encoding for the whole batch and all heads, expanded: its gradient sums over them
    one = torch.randn(1, 1, sk, d, device=cuda, requires_grad=True)
    x = q.clone().requires_grad_(True)
    o = cfa.cross_attention(x, one.expand(b, h, sk, d), v, 0.125)
    (dk,) = torch.autograd.grad(o, one, dout)
    full, size = ref.cross(q, one.expand(b, h, sk, d), v, 0.125, None, dout)
    near(o, full[0], size[0], "o")
    near(dk, full[2].sum((0, 1), keepdim=True), size[2].sum((0, 1), keepdim=True), "dk")
    # keys and values that are one tensor
    kv = k.clone().requires_grad_(True)
    (dkv,) = torch.autograd.grad(cfa.cross_attention(q, kv, kv, 0.125), kv, dout)
    full, size = ref.cross(q, k, k, 0.125, None, dout)
    near(dkv, full[2] + full[3], size[2] + size[3], "dkv")
    # a gradient that is itself a broadcast
    y = q.clone().requires_grad_(True)
    cfa.cross_attention(y, k, v, 0.125).sum().backward()
    full, size = ref.cross(q, k, v, 0.125, None, torch.ones(b, h, sq, d))
    near(y.grad, full[1], size[1], "dq")


@pytest.mark.parametrize("d", [32, 64, 128])
def test_gradient_against_differences(cuda, d):
    """Directional central differences of L = sum o w. Over eps = 2^-6 the third-order term is below
    eps^2 |u|^3-ish (2e-3 of the derivative at unit inputs and scale 1 / sqrt d), the outputs' own
    error 1e-6 |o| |w| / eps."""
    g = torch.Generator().manual_seed(d)
    q, k, v, w = (t.to(cuda) for t in make(2, 4, 2, 9, 11, d, None, seed=d))
    lengths = torch.tensor([11, 6], dtype=torch.int32, device=cuda)
    scale = 1.0 / math.sqrt(d)
    x = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(cfa.cross_attention(*x, scale, key_lengths=lengths), x, w)
    eps = 2.0 ** -6
    for i, name in enumerate("qkv"):
        u = torch.randn(x[i].shape, generator=g).to(cuda)
        loss = []
        for sgn in (1, -1):
            y = [t.detach() for t in x]
            y[i] = y[i] + sgn * eps * u
            # (requires_grad: the kernels of the training path)
            o = cfa.cross_attention(y[0].requires_grad_(True), *y[1:], scale, key_lengths=lengths)
            loss.append(float((o.detach().double() * w.double()).sum()))
        diff = (loss[0] - loss[1]) / (2 * eps)
        want = float((grads[i].double() * u.double()).sum())
        size = float(grads[i].double().norm() * math.sqrt(u.numel()))
        assert abs(diff - want) <= 2e-3 * size + 1e-6 * float(w.norm()) * 10 / eps, name


@pytest.mark.parametrize("scale", [0.0, -0.125, 4.0])
def test_scales(cuda, scale):
    check(cuda, 2, 2, 2, 70, 90, 64, [90, 33], scale=scale)


def test_empty(cuda):
    for b, h, hk, sq, sk in ((0, 2, 2, 3, 4), (2, 0, 0, 3, 4), (2, 2, 1, 0, 4), (2, 2, 1, 3, 0), (2, 2, 2, 0, 0)):
        x = [torch.ones(b, n, s, 64, device=cuda, requires_grad=True)
             for n, s in ((h, sq), (hk, sk), (hk, sk))]
        o = cfa.cross_attention(*x, 0.125)
        assert o.shape == (b, h, sq, 64) and not o.any()
        for g, t in zip(torch.autograd.grad(o.sum(), x), x):
            assert g.shape == t.shape and not g.any()
        with torch.no_grad():
            assert not cfa.cross_attention(*x, 0.125).any()
    cfa.check_status()


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("sq", [3, 70, 700])
def test_one_key_has_no_gradient(cuda, d, sq):
    """Its weight is one whatever the score: dQ and dK are zeros, not what is left of a cancellation."""
    _, _, o, (dq, dk, dv) = run(cuda, 2, 4, 2, sq, 130, d, [1, 130])
    assert not dq[0].any() and not dk[0].any() and dv[0, :, 0].any() and dq[1].any() and dk[1].any()
    _, _, o, (dq, dk, dv) = run(cuda, 2, 2, 2, sq, 1, d, None)
    assert not dq.any() and not dk.any() and dv.any()


def test_no_query_heads(cuda):
    """Key heads that no query reads: their gradients are zeros, whatever the memory held."""
    for h, sq in ((0, 3), (2, 0), (0, 0)):
        q = torch.ones(2, h, sq, 64, device=cuda, requires_grad=True)
        k, v = (torch.ones(2, 2, 70, 64, device=cuda, requires_grad=True) for _ in range(2))
        o = cfa.cross_attention(q, k, v, 0.125)
        used = torch.full((2, 70, 2, 2, 64), 7.0, device=cuda)
        del used
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.empty_like(o))
        assert dq.shape == q.shape and not dk.any() and not dv.any()
    cfa.check_status()


def test_graph_capture_and_streams(cuda):
    """A forward and backward captured once and replayed on new inputs; and on a side stream."""
    q, k, v, dout = (t.to(cuda) for t in make(2, 4, 2, 70, 300, 64, None))
    lengths = torch.tensor([300, 90], dtype=torch.int32, device=cuda)

    def step(q, k, v, dout):
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = cfa.cross_attention(*x, 0.125, key_lengths=lengths)
        return (o.detach(), *torch.autograd.grad(o, x, dout))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step(q, k, v, dout)
    torch.cuda.current_stream().wait_stream(s)
    want = step(q, k, v, dout)
    assert all(torch.equal(a, c) for a, c in zip(side, want))
    static = [t.clone() for t in (q, k, v, dout)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for t in static:
        t.mul_(0.5)
    lengths.copy_(torch.tensor([17, 0], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want = step(*static)
    assert all(torch.equal(a, c) for a, c in zip(out, want))
    cfa.check_status()


def test_training_step_with_rotary_and_projection(cuda):
    """The operators together, as an encoder-decoder layer's step: project, rotate, attend to the
    sequence itself, then to the encoding; every gradient against torch's in 64 bits."""
    b, s, sk, h, d = 2, 24, 40, 3, 64
    g = torch.Generator().manual_seed(3)
    hid = h * d
    x, enc = torch.randn(b, s, hid, generator=g), torch.randn(b, sk, hid, generator=g)
    w1, wq, wkv = (torch.randn(hid, n * hid, generator=g) / math.sqrt(hid) for n in (3, 1, 2))
    lens = torch.tensor([40, 13], dtype=torch.int32)
    freqs = 100.0 ** (-2.0 * torch.arange(d // 2, dtype=torch.float64) / d)

    def ours(x, enc, w1, wq, wkv):
        qkv = cfa.rotary_qkv(cfa.broadcast_matmul(x, w1), h, 7, freqs.to(cuda))
        y = cfa.fused_attention_qkv(qkv, h, 0.125, True)
        q = cfa.broadcast_matmul(y, wq).view(b, s, h, d).transpose(1, 2)
        k, v = cfa.broadcast_matmul(enc, wkv).view(b, sk, 2, h, d).permute(2, 0, 3, 1, 4)
        return cfa.cross_attention(q, k, v, 0.125, key_lengths=lens.to(cuda))

    def plain(x, enc, w1, wq, wkv):
        q, k, v = (x @ w1).view(b, s, 3, h, d).permute(2, 0, 3, 1, 4)
        angle = torch.arange(7, 7 + s, dtype=torch.float64)[:, None] * freqs
        c, sn = angle.cos(), angle.sin()
        turn = lambda t: torch.cat((t[..., :32] * c - t[..., 32:] * sn,  # noqa: E731
                                    t[..., 32:] * c + t[..., :32] * sn), -1)
        y = turn(q) @ turn(k).transpose(2, 3) * 0.125
        y = torch.softmax(y.masked_fill(torch.ones(s, s).triu(1).bool(), -math.inf), -1) @ v
        q = (y.transpose(1, 2).reshape(b, s, hid) @ wq).view(b, s, h, d).transpose(1, 2)
        k, v = (enc @ wkv).view(b, sk, 2, h, d).permute(2, 0, 3, 1, 4)
        y = q @ k.transpose(2, 3) * 0.125
        out = torch.arange(sk) >= lens[:, None, None, None]
        return torch.softmax(y.masked_fill(out, -math.inf), -1) @ v

    dout = torch.randn(b, h, s, d, generator=g)
    inputs = (x, enc, w1, wq, wkv)
    a = [t.to(cuda).requires_grad_(True) for t in inputs]
    c = [t.double().requires_grad_(True) for t in inputs]
    oa, oc = ours(*a), plain(*c)
    ga = torch.autograd.grad(oa, a, dout.to(cuda))
    gc = torch.autograd.grad(oc, c, dout.double())
    for got, want in zip((oa, *ga), (oc, *gc)):
        # five operators after one another, 1e-5 each
        assert (got.detach().cpu().double() - want.detach()).norm() <= 5 * BAND * want.detach().norm()
    cfa.check_status()

# SPDX-License-Identifier: MIT OR Apache-2.0
"""The paged cache: paged_append and paged_attention against the 64-bit formulas
(tests/formulas.py), over types, page sizes and orders, lengths, groups, and what a cache holds
where no result may look."""

import math

import pytest
import torch

import candle_fused_attn as cfa
import formulas as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F32, F32), (F32, F16), (F32, BF16), (F16, F16), (BF16, BF16)]
U = 2.0 ** -24


def band(q, k, v, scale, out, dtype):
    """How far an output may be off: with R = max |k| |q| scale over the rows, scores are off by (d +
    4) u R (d products in fp32; the tensor core's truncating windows of d / 16 steps stay within it)
    and the exponent's argument by 2 u of at most 25 (smaller p do not matter), 2^x by 4 u: p is off
    by a factor of 2 ((d + 4) R + 54) u both above and below the line; p's 16 bits for a 16-bit
    output add 2^-16; the sums of n terms in chunks add (n / 16 + 64) u. All of them times max |v|,
    then half a step of the output's type."""
    d, n = q.shape[-1], max(k.shape[1], 1)
    size = scale * q.abs().amax() * k.abs().sum(-1).amax() if k.numel() else 0.0
    rel = (2 * ((d + 4) * float(size) + 54) + n / 16 + 64) * U
    top = float(v.abs().amax()) if v.numel() else 0.0
    if dtype == F32:
        return rel * top
    return (rel + 2.0 ** -16) * top + torch.finfo(dtype).eps / 2 * out.abs() + 2.0 ** -25


def make(lens, h, hk, s, d, page, order, qt, kt, seed=0, fill=float("nan")):
    g = torch.Generator().manual_seed(seed)
    k = [torch.randn(hk, n, d, generator=g).to(kt) for n in lens]
    v = [torch.randn(hk, n, d, generator=g).to(kt) for n in lens]
    q = torch.randn(len(lens), h, s, d, generator=g).to(qt)
    return q, k, v, ref.paged(k, v, page, g, kt, order=order, fill=fill)


def check_attention(cuda, lens, h, hk, s, d, page, order, qt, kt, seed=0, scale=None, new=None):
    q, k, v, (kc, vc, table, lengths) = make(lens, h, hk, s, d, page, order, qt, kt, seed)
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    args = [t.to(cuda) for t in (q, kc, vc, table, lengths)]
    counts = None if new is None else torch.tensor(new, dtype=torch.int32, device=cuda)
    o = cfa.paged_attention(*args, scale, new_lengths=counts)
    cfa.check_status()
    assert o.shape == q.shape and o.dtype == qt and o.transpose(1, 2).is_contiguous()
    o = o.cpu().double()
    for i, n in enumerate(lens):
        m = s if new is None else new[i]
        seen = [n - m + j + 1 if j < m else 0 for j in range(s)]
        want = ref.attend(q[i].double(), k[i].double(), v[i].double(), scale, seen)
        err = (o[i] - want).abs()
        lim = band(q[i].double(), k[i].double(), v[i].double(), abs(scale), want, qt)
        assert bool((err <= lim).all()), f"sequence {i} of {n}: {err.max():.2e}"
        for j, c in enumerate(seen):
            if c <= 0:
                assert not o[i, :, j].any()
    return args, o


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("h,hk", [(1, 1), (6, 6), (8, 2), (9, 3), (16, 1), (20, 2)])
def test_types_dims_and_groups(cuda, qt, kt, d, h, hk):
    check_attention(cuda, [1, 0, 63, 64, 65, 200, 17], h, hk, 1, d, 16, "token", qt, kt, seed=d + h)


@pytest.mark.parametrize("qt,kt", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16)])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("order", ["token", "head"])
def test_pages(cuda, qt, kt, page, order):
    check_attention(cuda, [1, page, page + 1, 130, 333], 4, 2, 1, 64, page, order, qt, kt, seed=page)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("n", [1023, 1024, 1025, 2049, 4097, 8200, 20000])
def test_chunk_borders(cuda, qt, kt, n):
    """Lengths on both sides of where the chunk size changes."""
    check_attention(cuda, [n, 5, n - 1], 2, 1, 1, 64, 64, "token", qt, kt, seed=n)


@pytest.mark.parametrize("qt,kt", [(F32, F32), (BF16, BF16), (F32, F16)])
def test_very_long(cuda, qt, kt):
    """More than 256 chunks of 512: the chunks grow."""
    check_attention(cuda, [140_001], 2, 2, 1, 32, 256, "head", qt, kt, seed=1)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("s,h,hk", [(2, 2, 2), (5, 4, 2), (3, 6, 1), (40, 2, 1), (17, 9, 3)])
def test_several_new_tokens(cuda, qt, kt, s, h, hk):
    """Query i of s sees the keys up to its own; sequences shorter than s have rows that see none."""
    check_attention(cuda, [s, 1, 0, s + 1, 16, 90, 300], h, hk, s, 64, 16, "token", qt, kt, seed=s)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("s,h,hk", [(1, 3, 1), (1, 16, 2), (3, 3, 1), (2, 16, 2), (17, 1, 1), (4, 10, 1)])
def test_rows_of_a_key_head(cuda, qt, kt, d, s, h, hk):
    """3, 8, 9, 16, 17 and 40 query rows a key head: each kernel's first and last, and one row over."""
    check_attention(cuda, [333, 0, 1, 40, 1500, 16], h, hk, s, d, 24, "head", qt, kt, seed=s + h)
    check_attention(cuda, [64, 700], h, hk, s, d, 32, "token", qt, kt, seed=s)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_unseen_keys_of_many_rows_may_hold_anything(cuda, qt, kt, d):
    """As above for 24 rows a key head: the last token's key is infinite, its value NaN."""
    n, s, h = 45, 3, 8
    q, k, v, _ = make([n], h, 1, s, d, 16, "token", qt, kt, seed=19)
    k[0][:, n - 1] = math.inf
    v[0][:, n - 1] = math.nan
    kc, vc, table, lengths = ref.paged(k, v, 16, torch.Generator().manual_seed(1), kt)
    o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), 0.125)
    cfa.check_status()
    k0, v0 = (t[0][:, :n - 1].double() for t in (k, v))
    want = ref.attend(q[0].double(), k0, v0, 0.125, [n - 2, n - 1, 0])[:, :2]
    lim = band(q[0].double(), k0, v0, 0.125, want, qt)
    assert bool(((o[0].cpu().double()[:, :2] - want).abs() <= lim).all())


@pytest.mark.parametrize("qt,kt", [(F32, F32), (BF16, BF16)])
def test_padded_new_tokens(cuda, qt, kt):
    check_attention(cuda, [10, 70, 3, 64, 5], 4, 2, 4, 64, 16, "token", qt, kt,
                    new=[4, 1, 0, 3, 2])


@pytest.mark.parametrize("qt,kt", TYPES)
def test_unseen_keys_may_hold_anything(cuda, qt, kt):
    """A later token's key and value are infinite and NaN: earlier queries do not see them. (Rows
    past a length hold NaN in every test here.)"""
    n, s, d = 50, 3, 64
    q, k, v, _ = make([n], 4, 2, s, d, 16, "token", qt, kt, seed=9)
    k[0][:, n - 1] = math.inf
    v[0][:, n - 1] = math.nan
    kc, vc, table, lengths = ref.paged(k, v, 16, torch.Generator().manual_seed(1), kt)
    o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), 0.125)
    cfa.check_status()
    want = ref.attend(q[0].double(), k[0][:, :n - 1].double(), v[0][:, :n - 1].double(), 0.125,
                      [n - 2, n - 1, 0])
    err = (o[0].cpu().double() - want).abs()[:, :2]
    lim = band(q[0].double(), k[0][:, :n - 1].double(), v[0][:, :n - 1].double(), 0.125, want, qt)
    assert bool((err <= (lim if isinstance(lim, float) else lim[:, :2])).all())


@pytest.mark.parametrize("qt,kt", TYPES)
def test_large_and_small_scores(cuda, qt, kt):
    """Scores of hundreds (one key takes all), tiny queries, a zero and a negative scale."""
    lens, d = [200, 77], 64
    g = torch.Generator().manual_seed(12)
    for qs, scale in ((30.0, 0.5), (1e-6, 0.125), (1.0, 0.0), (1.0, -0.125)):
        q = (torch.randn(2, 2, 1, d, generator=g) * qs).to(qt)
        k = [torch.randn(2, n, d, generator=g).to(kt) for n in lens]
        v = [torch.randn(2, n, d, generator=g).to(kt) for n in lens]
        kc, vc, table, lengths = ref.paged(k, v, 16, g, kt)
        o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), scale)
        for i in range(2):
            want = ref.attend(q[i].double(), k[i].double(), v[i].double(), scale, [lens[i]])
            lim = band(q[i].double(), k[i].double(), v[i].double(), abs(scale), want, qt)
            assert bool(((o[i].cpu().double() - want).abs() <= lim).all())


def test_wide_range_fp32_queries_over_fp16(cuda):
    """fp32 queries past fp16's range, up and down: the parts go under a power of two per row."""
    g = torch.Generator().manual_seed(13)
    for size in (1e-30, 1e-6, 1e6, 1e30):
        q = torch.randn(1, 2, 1, 64, generator=g) * size
        k, v = [torch.randn(2, 40, 64, generator=g).half()], [torch.randn(2, 40, 64, generator=g).half()]
        kc, vc, table, lengths = ref.paged(k, v, 16, g, F16)
        scale = 0.125 / size
        o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), scale)
        want = ref.attend(q[0].double(), k[0].double(), v[0].double(), scale, [40])
        lim = band(q[0].double(), k[0].double(), v[0].double(), scale, want, F32)
        assert bool(((o[0].cpu().double() - want).abs() <= lim).all())


def test_wide_range_of_many_rows(cuda):
    """The same for 12 rows, each of a size of its own."""
    g = torch.Generator().manual_seed(14)
    size = 10.0 ** torch.linspace(-25, 25, 12)[None, :, None, None]
    q = torch.randn(1, 12, 1, 64, generator=g) * size
    k, v = [torch.randn(1, 40, 64, generator=g).half()], [torch.randn(1, 40, 64, generator=g).half()]
    kc, vc, table, lengths = ref.paged(k, v, 16, g, F16)
    for i, scale in ((0, 1e24), (6, 0.01), (11, 1e-26)):
        o = cfa.paged_attention(*(t.to(cuda) for t in (q, kc, vc, table, lengths)), scale)
        row = q[0, i:i + 1].double()
        want = ref.attend(row, k[0].double(), v[0].double(), scale, [40])
        lim = band(row, k[0].double(), v[0].double(), scale, want, F32)
        assert bool(((o[0, i].cpu().double() - want[0]).abs() <= lim).all())


def test_bitwise_reruns_batches_and_shared_pages(cuda):
    """A sequence's result is its own: alone, in a batch, with its pages shared with another (the same
    prefix twice), and again."""
    for (qt, kt), h in ((t, h) for t in TYPES for h in (8, 24)):
        args, _ = check_attention(cuda, [900, 31, 5000, 1], h, 2, 1, 64, 16, "token", qt, kt)
        q, kc, vc, table, lengths = args
        o = cfa.paged_attention(*args, 0.125)
        assert torch.equal(o, cfa.paged_attention(*args, 0.125))
        for i in range(4):
            one = cfa.paged_attention(q[i:i + 1], kc, vc, table[i:i + 1], lengths[i:i + 1], 0.125)
            assert torch.equal(one[0], o[i])
        twice = [2, 2, 0]
        o2 = cfa.paged_attention(q[[2, 2, 0]], kc, vc, table[twice], lengths[twice], 0.125)
        assert torch.equal(o2[0], o[2]) and torch.equal(o2[1], o[2]) and torch.equal(o2[2], o[0])


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_a_wider_table_changes_nothing(cuda, qt, kt, d):
    """Room for more pages (and with it another way of joining the chunks): the same bits."""
    args, _ = check_attention(cuda, [5000, 31, 2000, 600], 4, 2, 1, d, 16, "token", qt, kt)
    q, kc, vc, table, lengths = args
    want = cfa.paged_attention(*args, 0.125)
    for width in (2000, 20000):
        wide = torch.full((4, width), -1, dtype=torch.int32, device=cuda)
        wide[:, :table.shape[1]] = table
        assert torch.equal(cfa.paged_attention(q, kc, vc, wide, lengths, 0.125), want)
    cfa.check_status()


def test_strided_and_unaligned_queries(cuda):
    args, _ = check_attention(cuda, [100, 40], 4, 2, 1, 64, 16, "token", F32, F32)
    q, rest = args[0], args[1:]
    want = cfa.paged_attention(q, *rest, 0.125)
    wide = torch.zeros(2, 4, 1, 70, device=cuda)
    for at in (0, 1, 2):
        wide[..., at:at + 64] = q
        assert torch.equal(cfa.paged_attention(wide[..., at:at + 64], *rest, 0.125), want)
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(cfa.paged_attention(swapped, *rest, 0.125), want)


@pytest.mark.parametrize("qt,kt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("hk,h,s,d,rot,page,order", [
    (2, 4, 1, 64, 64, 16, "token"), (1, 1, 5, 32, 32, 8, "head"), (3, 6, 33, 128, 64, 24, "token"),
    (2, 2, 7, 40, 20, 1, "token"), (4, 0, 3, 64, 0, 64, "head"), (8, 64, 2, 128, 128, 16, "token")])
def test_append(cuda, qt, kt, interleaved, hk, h, s, d, rot, page, order):
    """Every slot of the new tokens, nothing else, and the rotated queries."""
    g = torch.Generator().manual_seed(page + s)
    before = [0, 5, page, 77]
    new = [s, s, 0, max(s - 1, 0)]
    lens = [x + n for x, n in zip(before, new)]
    old = [torch.randn(hk, n, d, generator=g) for n in lens]
    kc, vc, table, lengths = ref.paged(old, old, page, g, kt, order=order, fill=3.0)
    q, k, v = (torch.randn(4, n, s, d, generator=g).to(qt) for n in (h, hk, hk))
    freqs = None if rot == 0 else 500.0 ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    dk, dvc = kc.clone().to(cuda), vc.clone().to(cuda)
    if order == "head":  # keep the pool's order
        dk, dvc = (t.transpose(1, 2).contiguous().to(cuda).transpose(1, 2) for t in (kc, vc))
    out = cfa.paged_append(k.to(cuda), v.to(cuda), dk, dvc, table.to(cuda), lengths.to(cuda),
                           q=q.to(cuda) if h else None,
                           freqs=None if freqs is None else freqs.to(cuda), amplitude=1.1,
                           interleaved=interleaved,
                           new_lengths=torch.tensor(new, dtype=torch.int32, device=cuda))
    cfa.check_status()
    assert (out is None) == (h == 0)
    none = torch.zeros(0, dtype=torch.float64)
    fr = none if freqs is None else freqs
    kb = ref.rotate_band(k, fr, 1.1, interleaved, kt)
    qb = ref.rotate_band(q, fr, 1.1, interleaved, qt)
    want_v = vc.clone()
    touched = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for i in range(4):
        pos = torch.arange(before[i], before[i] + new[i])
        kr = ref.rotate(k[i:i + 1, :, :new[i]], pos, fr, 1.1, interleaved)[0]
        for j in range(new[i]):
            pg, r = int(table[i, (before[i] + j) // page]), (before[i] + j) % page
            touched[pg, r] = True
            err = (dk[pg, r].cpu().double() - kr[:, j]).abs()
            assert bool((err <= kb[i, :, j]).all())
            want_v[pg, r] = v[i, :, j].to(kt)
        if h:
            qr = ref.rotate(q[i:i + 1, :, :new[i]], pos, fr, 1.1, interleaved)[0]
            got = out[i].cpu().double()
            assert bool(((got[:, :new[i]] - qr).abs() <= qb[i, :, :new[i]]).all())
            assert not got[:, new[i]:].any()
    assert torch.equal(dvc.cpu(), want_v)
    assert torch.equal(dk.cpu()[~touched], kc[~touched])


def test_append_unaligned_and_strided(cuda):
    """Odd offsets and a fused projection's views take the narrow accesses: the same bits."""
    g = torch.Generator().manual_seed(2)
    for kt in (F32, BF16):
        old = [torch.randn(2, 20, 64, generator=g) for _ in range(3)]
        kc, vc, table, lengths = ref.paged(old, old, 16, g, kt, fill=0.0)
        table, lengths = table.to(cuda), lengths.to(cuda)
        freqs, _ = cfa.rotary_frequencies(64, device=cuda)
        qkv = torch.randn(3, 4, 8, 65, generator=g).to(cuda).to(kt)
        got = []
        for x in (qkv[..., 1:], qkv[..., 1:].contiguous()):
            q, k, v = (t.transpose(1, 2) for t in x.split((4, 2, 2), 2))
            a, b = kc.to(cuda), vc.to(cuda)
            got.append((cfa.paged_append(k, v, a, b, table, lengths, q=q, freqs=freqs), a, b))
        for x, y in zip(*got):
            assert torch.equal(x, y)


def test_bad_pages_are_reported_and_skipped(cuda):
    """A page id outside the cache (the index checks run first on the CPU: test_operators.py): the
    other keys are attended, nothing is written, the next call raises, and calls go on."""
    q, k, v, (kc, vc, table, lengths) = make([40, 40], 2, 2, 1, 64, 16, "token", F32, F32, fill=0.0)
    table[1, 1] = 1000
    args = [t.to(cuda) for t in (q, kc, vc, table, lengths)]
    o = cfa.paged_attention(*args, 0.125)
    with pytest.raises(cfa.FusedAttentionError, match="page id"):
        cfa.check_status()
    keep = list(range(16)) + list(range(32, 40))
    for i, rows in ((0, list(range(40))), (1, keep)):
        want = ref.attend(q[i].double(), k[i][:, rows].double(), v[i][:, rows].double(), 0.125,
                          [len(rows)])
        assert (o[i].cpu().double() - want).abs().max() < 1e-4
    kd, vd = args[1].clone(), args[2].clone()
    new = torch.randn(2, 2, 1, 64, device=cuda)
    args[4] -= 20  # the new token of sequence 1 sits on the bad page
    cfa.paged_append(new, new, kd, vd, args[3], args[4])
    with pytest.raises(cfa.FusedAttentionError, match="page id"):
        cfa.check_status()
    changed = (kd != args[1]).any(-1).any(-1).nonzero().tolist()
    assert changed == [[int(table[0, 1]), 3]]
    args[4] += 100  # a length past the table: cut there, and reported
    cfa.paged_attention(*args, 0.125)
    with pytest.raises(cfa.FusedAttentionError, match="length past"):
        cfa.check_status()
    args[3][1, 1] = args[3][0, 1]
    args[4].fill_(40)
    cfa.paged_attention(*args, 0.125)
    cfa.check_status()


def test_decoding_steps_in_a_graph(cuda):
    """A decoding loop -- lengths, append, attend -- captured once and replayed: each step's output is
    that of plain attention over the tokens so far, the two graphs on one cache do not disturb each
    other, and eager steps give the same bits."""
    b, h, hk, d, page, steps = 3, 4, 2, 64, 4, 9
    g = torch.Generator().manual_seed(21)
    freqs, _ = cfa.rotary_frequencies(d, device=cuda)
    qkv = torch.randn(steps, b, 1, h + 2 * hk, d, generator=g).to(cuda)
    table = torch.randperm(b * 3, generator=g).int().view(b, 3).to(cuda)

    def state():
        return (torch.zeros(3 * b, page, hk, d, device=cuda), torch.zeros(3 * b, page, hk, d, device=cuda),
                torch.zeros(b, dtype=torch.int32, device=cuda), qkv[0].clone())

    def step(kc, vc, lengths, x):
        lengths += 1
        q, k, v = (t.transpose(1, 2) for t in x.split((h, hk, hk), 2))
        q = cfa.paged_append(k, v, kc, vc, table, lengths, q=q, freqs=freqs)
        return cfa.paged_attention(q, kc, vc, table, lengths, 0.125)

    eager, outs = state(), []
    for t in range(steps):
        eager[3].copy_(qkv[t])
        outs.append(step(*eager).clone())
    for t in (0, 4, steps - 1):
        seq = qkv[:t + 1].squeeze(2)  # [t + 1, b, heads, d]
        for i in range(b):
            x = seq[:, i].transpose(0, 1)[None]
            pos = torch.arange(t + 1)
            kr = ref.rotate(x[:, h:h + hk], pos, freqs)[0]
            qr = ref.rotate(x[:, :h, t:], pos[t:], freqs)[0]
            want = ref.attend(qr, kr, x[0, h + hk:].cpu().double(), 0.125, [t + 1])
            # rotated operands are 9 u off each; 5e-5 is far above that and below any wrong key
            assert (outs[t][i].cpu().double() - want).abs().max() < 5e-5
    one, two = state(), state()
    graphs = []
    for s in (one, two):
        warm = [x.clone() for x in s]
        step(*warm)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*s)
        graphs.append((graph, out))
    for t in range(steps):
        for s, (graph, out) in zip((one, two), graphs):
            s[3].copy_(qkv[t])
            graph.replay()
        for _, out in graphs:
            assert torch.equal(out, outs[t])
    cfa.check_status()


def test_two_streams_at_once(cuda):
    args, _ = check_attention(cuda, [3000, 100], 8, 2, 1, 64, 16, "token", BF16, BF16)
    want = cfa.paged_attention(*args, 0.125)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(cfa.paged_attention(*args, 0.125))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


def test_empty(cuda):
    kc = torch.zeros(4, 16, 2, 64, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    o = cfa.paged_attention(torch.zeros(0, 2, 1, 64, device=cuda), kc, kc, torch.zeros(0, 3, **i32),
                            torch.zeros(0, **i32), 1.0)
    assert o.shape == (0, 2, 1, 64)
    # no page at all: nothing to see
    o = cfa.paged_attention(torch.ones(2, 2, 1, 64, device=cuda), kc, kc, torch.zeros(2, 0, **i32),
                            torch.zeros(2, **i32), 1.0)
    assert o.shape == (2, 2, 1, 64) and not o.any()
    x = torch.ones(2, 2, 0, 64, device=cuda)
    cfa.paged_append(x, x, kc, kc.clone(), torch.zeros(2, 1, **i32), torch.zeros(2, **i32))
    assert not kc.any()
    cfa.check_status()

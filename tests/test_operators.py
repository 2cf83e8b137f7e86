# SPDX-License-Identifier: MIT OR Apache-2.0
"""The operators beside the fused attention on the CPU: what their entry points refuse before
anything reaches a device, the workspace sizes, the frequencies, and the paged cache's index
arithmetic (a page id outside the pool never becomes an address)."""

import math
import random

import pytest
import torch

import candle_fused_attn as cfa
from candle_fused_attn import _abi

FAKE = 1 << 20  # a 16-byte aligned non-null "device pointer" no check dereferences
S3 = (64 * 64, 64, 64)


# --- the C ABI ------------------------------------------------------------------------------------

def cross_fwd(q=FAKE, k=FAKE, o=FAKE, dims=(2, 4, 2, 8, 9, 64), st=S3):
    return _abi.cross_fwd(q, st, k, st, k, st, None, o, FAKE, *dims, 0.1, None)


def test_cross_forward_arguments():
    assert cross_fwd(dims=(-1, 4, 2, 8, 9, 64)) == _abi.CFA_ERR_SHAPE
    assert cross_fwd(dims=(2, 4, 2, 8, 9, 48)) == _abi.CFA_ERR_HEAD_DIM
    assert cross_fwd(dims=(2, 4, 3, 8, 9, 64)) == _abi.CFA_ERR_HEADS
    assert cross_fwd(dims=(2, 4, 0, 8, 9, 64)) == _abi.CFA_ERR_HEADS
    assert cross_fwd(dims=(1 << 20, 1 << 10, 1 << 10, 1 << 10, 9, 64)) == _abi.CFA_ERR_OVERFLOW
    assert cross_fwd(dims=(1 << 16, 1 << 10, 1, 1, 1 << 20, 64)) == _abi.CFA_ERR_OVERFLOW
    assert cross_fwd(q=None) == _abi.CFA_ERR_NULL and cross_fwd(k=None) == _abi.CFA_ERR_NULL
    assert cross_fwd(q=FAKE + 4) == _abi.CFA_ERR_ALIGNMENT
    assert cross_fwd(k=FAKE + 8) == _abi.CFA_ERR_ALIGNMENT
    assert cross_fwd(st=(64, 64, 66)) == _abi.CFA_ERR_ALIGNMENT
    for empty in ((0, 4, 2, 8, 9, 64), (2, 0, 0, 8, 9, 64), (2, 4, 2, 0, 9, 64)):
        assert cross_fwd(q=None, k=None, o=None, dims=empty) == _abi.CFA_OK


def test_cross_backward_arguments():
    dims = (2, 4, 2, 8, 9, 64)
    need = _abi.cross_bwd_workspace_bytes(*dims)

    def call(q=FAKE, dq=FAKE, ws=FAKE, nbytes=need, dims=dims):
        return _abi.cross_bwd(q, S3, FAKE, S3, FAKE, S3, None, FAKE, FAKE, FAKE, S3, dq, FAKE, ws,
                              nbytes, *dims, 0.1, None)

    assert call(nbytes=need - 1) == _abi.CFA_ERR_WORKSPACE
    assert call(ws=FAKE + 16) == _abi.CFA_ERR_WORKSPACE
    assert call(ws=None) == _abi.CFA_ERR_NULL and call(dq=None) == _abi.CFA_ERR_NULL
    assert call(q=FAKE + 4) == _abi.CFA_ERR_ALIGNMENT
    assert call(dims=(2, 3, 2, 8, 9, 64)) == _abi.CFA_ERR_HEADS
    assert call(dims=(2, 4, 2, 8, -9, 64)) == _abi.CFA_ERR_SHAPE
    assert call(dims=(2, 4, 2, 8, 9, 16)) == _abi.CFA_ERR_HEAD_DIM
    assert call(dims=(0, 4, 2, 8, 9, 64)) == _abi.CFA_OK
    assert call(dims=(2, 4, 2, 0, 0, 64)) == _abi.CFA_OK


def test_cross_backward_workspace():
    """D and the turn counters always, and a dK, dV a part where the query tiles are cut into parts; the
    fast size adds the dQ partials, one a key block (of 128; of 64 at head dim 128), up to 4 GB."""
    size, fast = _abi.cross_bwd_workspace_bytes, _abi.cross_bwd_workspace_bytes_fast
    for fn in (size, fast):
        assert fn(0, 4, 2, 8, 9, 64) == 256 and fn(2, 4, 3, 8, 9, 64) == 256
    for d, kb in ((32, 128), (64, 128), (128, 64)):
        b, h, sq = 4, 37, 200  # 37 key heads, at least 16 key blocks: one part
        plain = 256 + b * h * 4 * 4 + b * h * sq * 4
        most = (4 << 30) // (b * h * sq * d * 4)
        for n in (16, 17, most):
            least = size(b, h, h, sq, n * kb, d)
            assert plain <= least <= plain + 1024
            assert fast(b, h, h, sq, n * kb, d) - least == n * b * h * sq * d * 4
        assert fast(b, h, h, sq, most * kb + 1, d) == size(b, h, h, sq, most * kb + 1, d)
    # more queries x key blocks than 2^63 bytes of partials: none
    huge = (1, 1, 1, 2**31 - 2000, 900_000_000, 128)
    assert size(*huge) > 2**32 and fast(*huge) == size(*huge)
    # 2 key blocks of one key head over 63 query tiles: 7 parts, each with a dK and dV of its own
    parts = 7 * 200 * 2 * 64 * 4
    whole = size(1, 8, 8, 500, 200, 64)  # 16 key blocks over 8 tiles each: one part
    assert size(1, 8, 1, 500, 200, 64) - parts == whole


def test_few_rows_arguments():
    dims = (2, 4, 2, 1, 900, 64)
    need = _abi.cross_few_workspace_bytes(2, 4, 1, 900, 64)
    assert need == 2 * 4 * 4 * 66 * 4  # four chunks of 256
    assert _abi.cross_few_workspace_bytes(2, 4, 1, 256, 64) == 0  # one chunk: nothing to join

    def call(q=FAKE, ws=FAKE, nbytes=need, dims=dims):
        return _abi.cross_few(q, S3, FAKE, S3, FAKE, S3, None, FAKE, None, ws, nbytes, *dims, 0.1,
                              None)

    assert call(nbytes=need - 1) == _abi.CFA_ERR_WORKSPACE
    assert call(ws=FAKE + 4) == _abi.CFA_ERR_WORKSPACE and call(ws=None) == _abi.CFA_ERR_NULL
    assert call(q=FAKE + 4) == _abi.CFA_ERR_ALIGNMENT
    assert call(dims=(2, 4, 3, 1, 900, 64)) == _abi.CFA_ERR_HEADS
    assert call(dims=(2, 4, 2, 0, 900, 64), q=None) == _abi.CFA_OK


def test_rotary_arguments():
    def call(x=FAKE, dtype=_abi.CFA_F32, pos=None, pos_bytes=0, freqs=FAKE, rotated=4,
             dims=(2, 4, 8, 64), rot=64):
        b, h, s, d = dims
        return _abi.rotary(x, S3, FAKE, S3, dtype, pos, pos_bytes, (8, 1), 0, freqs, 1.0, b, h,
                           rotated, s, d, rot, False, False, None)

    assert call(rot=63) == _abi.CFA_ERR_ROTARY and call(rot=66) == _abi.CFA_ERR_ROTARY
    assert call(rotated=5) == _abi.CFA_ERR_SHAPE and call(dims=(2, 4, -1, 64)) == _abi.CFA_ERR_SHAPE
    assert call(dims=(2, 4, 8, 1026)) == _abi.CFA_ERR_HEAD_DIM
    assert call(dtype=3) == _abi.CFA_ERR_TYPE and call(pos=FAKE, pos_bytes=2) == _abi.CFA_ERR_TYPE
    assert call(x=None) == _abi.CFA_ERR_NULL and call(freqs=None) == _abi.CFA_ERR_NULL
    assert call(dims=(1 << 20, 4, 1 << 20, 64)) == _abi.CFA_ERR_OVERFLOW
    assert call(dims=(0, 4, 8, 64), x=None) == _abi.CFA_OK


def append(q=FAKE, k=FAKE, types=(_abi.CFA_F32, _abi.CFA_BF16), pages=9, page=16, table=FAKE, width=3,
           lengths=FAKE, freqs=FAKE, dims=(2, 4, 2, 1, 64, 64)):
    return _abi.paged_append(q, S3, FAKE, S3, k, S3, FAKE, S3, types[0], FAKE, S3, FAKE, S3, types[1],
                             pages, page, table, width, width, lengths, None, freqs, 1.0, *dims, False,
                             None)


def test_append_arguments():
    assert append(types=(_abi.CFA_BF16, _abi.CFA_F32)) == _abi.CFA_ERR_TYPE
    assert append(types=(_abi.CFA_BF16, _abi.CFA_F16)) == _abi.CFA_ERR_TYPE
    assert append(types=(7, 7)) == _abi.CFA_ERR_TYPE
    assert append(page=0) == _abi.CFA_ERR_SHAPE and append(pages=-1) == _abi.CFA_ERR_SHAPE
    assert append(dims=(2, 4, 2, 1, 64, 65)) == _abi.CFA_ERR_ROTARY
    assert append(k=None) == _abi.CFA_ERR_NULL and append(lengths=None) == _abi.CFA_ERR_NULL
    assert append(table=None) == _abi.CFA_ERR_NULL and append(freqs=None) == _abi.CFA_ERR_NULL
    assert append(dims=(1 << 20, 4, 2, 1 << 20, 64, 64)) == _abi.CFA_ERR_OVERFLOW
    assert append(dims=(2, 4, 2, 0, 64, 64), k=None) == _abi.CFA_OK


def test_paged_attention_arguments():
    need = _abi.paged_attention_workspace_bytes(2, 4, 1, 3 * 640, 64, _abi.CFA_BF16)
    assert need == 2 * 4 * 4 * 66 * 4  # four chunks of 512

    def call(q=FAKE, types=(_abi.CFA_F32, _abi.CFA_BF16), cache=FAKE, page=640, width=3, table=FAKE,
             lengths=FAKE, ws=FAKE, nbytes=need, dims=(2, 4, 2, 1, 64), st=S3):
        return _abi.paged_attention(q, S3, types[0], cache, st, cache, st, types[1], 9, page, table,
                                    width, width, lengths, None, FAKE, ws, nbytes, *dims, 0.1, None)

    assert call(types=(_abi.CFA_F16, _abi.CFA_BF16)) == _abi.CFA_ERR_TYPE
    assert call(dims=(2, 4, 3, 1, 64)) == _abi.CFA_ERR_HEADS
    assert call(dims=(2, 4, 2, 1, 80)) == _abi.CFA_ERR_HEAD_DIM
    assert call(page=0) == _abi.CFA_ERR_SHAPE
    assert call(page=1 << 20, width=1 << 12) == _abi.CFA_ERR_OVERFLOW
    for name in ("q", "cache", "table", "lengths", "ws"):
        assert call(**{name: None}) == _abi.CFA_ERR_NULL
    assert call(cache=FAKE + 8) == _abi.CFA_ERR_ALIGNMENT
    assert call(st=(4096, 64, 60)) == _abi.CFA_ERR_ALIGNMENT  # 16-bit rows: multiples of 8
    assert call(nbytes=need - 1) == _abi.CFA_ERR_WORKSPACE
    assert call(dims=(0, 4, 2, 1, 64), q=None) == _abi.CFA_OK


def test_statuses_have_words():
    for code in (_abi.CFA_ERR_PAGE, _abi.CFA_ERR_TYPE, _abi.CFA_ERR_HEADS, _abi.CFA_ERR_ROTARY):
        assert _abi.strerror(code).startswith("fused_attention:")
        assert "unknown" not in _abi.strerror(code)


# --- the chunks of a sequence, as csrc/split_attn.cu cuts them ---------------------------------------

def chunk(n, tile):
    """16 tiles up to 16 chunks, 32 up to 256, then powers of two that keep them 256."""
    if n <= 256 * tile:
        return 16 * tile
    c = 32 * tile
    while n > 256 * c:
        c *= 2
    return c


@pytest.mark.parametrize("d,kv,tile", [(32, _abi.CFA_F32, 32), (64, _abi.CFA_F32, 16),
                                       (128, _abi.CFA_F32, 8), (32, _abi.CFA_F16, 32),
                                       (64, _abi.CFA_BF16, 32), (128, _abi.CFA_F16, 16)])
def test_workspace_holds_every_length_below_its_largest(d, kv, tile):
    """The workspace is sized for the longest sequence; a shorter one can have more chunks than it
    (its chunks are smaller) and must fit all the same."""
    most, r = 0, random.Random(1)
    lengths = sorted({*range(1, 9000), *(r.randint(9000, 4_000_000) for _ in range(3000)),
                      *(x + y for x in (1 << k for k in range(8, 31)) for y in (-1, 0, 1))})
    for n in lengths:
        most = max(most, -(-n // chunk(n, tile)))
        got = _abi.paged_attention_workspace_bytes(1, 1, 1, n, d, kv) // ((d + 2) * 4) or 1
        assert got >= most, n
    assert most <= 256


def test_page_lookup_never_leaves_the_pool():
    """The append's and the attention's index arithmetic over every kind of table entry and length:
    an address is formed only from a page id in the pool, a row in the page and a table entry that
    exists."""
    r = random.Random(2)
    for _ in range(2000):
        page, width, pages = r.randint(1, 64), r.randint(1, 9), r.randint(1, 20)
        table = [r.choice([r.randrange(pages), -1, pages, 2 ** 31 - 1, -2 ** 31]) for _ in range(width)]
        length = r.choice([r.randint(-5, page * width + 70), 0, page * width])
        cut = min(max(length, 0), page * width)  # what the attention reads of it
        for key in range(0, cut, r.randint(1, 7)):
            assert 0 <= key // page < width and 0 <= key - key // page * page < page
        n = r.randint(0, 5)
        for i in range(n):  # the append's tokens
            at = length - n + i
            if at < 0:
                continue
            lp = at // page
            pg = table[lp] if lp < width else -1
            if 0 <= pg < pages:
                assert 0 <= pg * page + at - lp * page < pages * page


# --- the Python layer -----------------------------------------------------------------------------

def raises(match):
    return pytest.raises(cfa.FusedAttentionError, match=match)


def test_cross_attention_refuses():
    q, k = torch.zeros(2, 4, 3, 64), torch.zeros(2, 2, 5, 64)
    with raises("CUDA tensors required"):
        cfa.cross_attention(q, k, k, 0.125)
    with raises("f32 only"):
        cfa.cross_attention(q.half(), k.half(), k.half(), 0.125)
    with raises("no multiple"):
        cfa.cross_attention(q, torch.zeros(2, 3, 5, 64), torch.zeros(2, 3, 5, 64), 0.125)
    with raises("expected, got"):
        cfa.cross_attention(q, k, k[:, :, :4], 0.125)
    with raises("expected, got"):
        cfa.cross_attention(q, k[:1], k[:1], 0.125)
    with raises("head_dim"):
        cfa.cross_attention(q[..., :48], k[..., :48], k[..., :48], 0.125)


def test_rotary_refuses():
    x = torch.zeros(2, 3, 4, 8)
    f = torch.ones(4, dtype=torch.float64)
    with raises("CUDA tensors required"):
        cfa.rotary(x, 0, f)
    with raises("float64"):
        cfa.rotary(x, 0, f.float())
    with raises("turn 10 dims"):
        cfa.rotary(x, 0, torch.ones(5, dtype=torch.float64))
    with raises("f32, f16 or bf16"):
        cfa.rotary(x.double(), 0, f)
    with raises(r"\[b, h, s, d\]"):
        cfa.rotary(x[0], 0, f)
    with raises("not 3 x 5 heads"):
        cfa.rotary_qkv(torch.zeros(2, 4, 72), 5, 0, f)
    with raises("x must be a tensor"):
        cfa.rotary([1.0], 0, f)
    with pytest.raises(TypeError):
        cfa.rotary(x, 0.5, f)
    with pytest.raises(OverflowError):
        cfa.rotary(x, 1 << 63, f)
    with pytest.raises(TypeError):
        cfa.rotary(x, 0, f, amplitude="1")
    with raises("freqs: has no backward"):
        cfa.rotary(x, 0, f.clone().requires_grad_(True))


def test_frequencies():
    f, a = cfa.rotary_frequencies(8, device="cpu")
    assert a == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64))
    lin, a = cfa.rotary_frequencies(8, scaling="linear", factor=4.0, device="cpu")
    assert a == 1.0 and torch.allclose(lin, f / 4)
    ntk, _ = cfa.rotary_frequencies(8, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and torch.allclose(ntk[-1], f[-1] / 4)
    yarn, a = cfa.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=4096, device="cpu")
    full = cfa.rotary_frequencies(64, device="cpu")[0]
    turns = 4096 * full / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], full[turns >= 32])
    assert torch.allclose(yarn[turns <= 1], full[turns <= 1] / 4)
    mid = (turns > 1) & (turns < 32)
    assert bool(((yarn[mid] < full[mid]) & (yarn[mid] > full[mid] / 4)).all()) and mid.any()
    assert a == pytest.approx(0.1 * math.log(4) + 1)
    with raises("even rotary"):
        cfa.rotary_frequencies(7, device="cpu")
    with raises("original_length"):
        cfa.rotary_frequencies(8, scaling="yarn", factor=2.0, device="cpu")
    with raises("unknown scaling"):
        cfa.rotary_frequencies(8, scaling="log", device="cpu")
    with raises("positive"):
        cfa.rotary_frequencies(8, factor=0.0, scaling="linear", device="cpu")


def paged(**kw):
    a = dict(q=torch.zeros(2, 4, 1, 64), kc=torch.zeros(3, 16, 2, 64), vc=None,
             table=torch.zeros(2, 3, dtype=torch.int32), lengths=torch.zeros(2, dtype=torch.int32),
             new=None)
    a.update(kw)
    if a["vc"] is None:
        a["vc"] = a["kc"]
    return a


def attend(**kw):
    a = paged(**kw)
    return cfa.paged_attention(a["q"], a["kc"], a["vc"], a["table"], a["lengths"], 0.1,
                               new_lengths=a["new"])


def append_py(**kw):
    a = paged(**kw)
    k = a.get("k", torch.zeros(2, 2, 1, 64))
    return cfa.paged_append(k, a.get("v", k), a["kc"], a["vc"], a["table"], a["lengths"], q=a["q"],
                            freqs=a.get("freqs"), new_lengths=a["new"])


def test_paged_calls_refuse():
    for call in (attend, append_py):
        with raises("CUDA tensors required"):
            call()
        with raises("over a cache of their type"):
            call(kc=torch.zeros(3, 16, 2, 64).double())
        with raises("caches"):
            call(vc=torch.zeros(3, 8, 2, 64))
        with raises("at least one row"):
            call(kc=torch.zeros(3, 0, 2, 64))
        with raises("last dimension"):
            call(kc=torch.zeros(3, 16, 2, 128)[..., ::2])
        with raises("page_table"):
            call(table=torch.zeros(2, 3, dtype=torch.int64))
        with raises("page_table"):
            call(table=torch.zeros(1, 3, dtype=torch.int32))
        with raises("lengths"):
            call(lengths=torch.zeros(2, dtype=torch.int64))
        with raises("new_lengths"):
            call(new=torch.zeros(3, dtype=torch.int32))
    with raises("of their type"):
        attend(q=torch.zeros(2, 4, 1, 64).half())
    with raises("no multiple"):
        attend(q=torch.zeros(2, 3, 1, 64))
    with raises("head_dim"):
        attend(q=torch.zeros(2, 4, 1, 48), kc=torch.zeros(3, 16, 2, 48))
    with raises("k and v"):
        append_py(k=torch.zeros(2, 2, 1, 64), v=torch.zeros(2, 2, 2, 64))
    with raises("of k's type"):
        append_py(q=torch.zeros(2, 4, 2, 64))
    with raises("CUDA|float64"):
        append_py(freqs=torch.ones(32))

# SPDX-License-Identifier: MIT OR Apache-2.0
"""The operators beside the fused attention, as programs call them, with their plain forms.

A case names an operator and its sizes. `prepare` makes a caller's inputs, `run` makes the call --
the plain form (elementary torch operations in 32 bits), or, where `own` is true, this package's
operator -- and `exact` computes the same from the definition in 64 bits.

- "cross":  cross_attention, an encoder's states of another length (padded batches by key lengths)
- "rotary": rotary, the position rotation of queries or keys
- "append": paged_append, new tokens into a paged cache with the rotation on the way
- "attend": paged_attention, the new tokens' attention over the paged cache
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parents[1] / "candle-fused-attn_b200"


def _cfa():
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    import candle_fused_attn
    return candle_fused_attn


def listed():
    return [
        # Queries of one new token a sequence, rotated before they attend: latency alone.
        dict(name="rotary_token", op="rotary", b=64, h=6, s=1, d=64, rot=64, layout="half",
             dtype="float32", backward=False, fused=False, start=1000, factor=1.0),
        # The training step's queries at the canvas shape, read out of the fused projection.
        dict(name="rotary_train", op="rotary", b=64, h=6, s=240, d=64, rot=64, layout="half",
             dtype="float32", backward=True, fused=True, start=0, factor=1.0),
        # A long 16-bit prompt with interleaved pairs in half of each head, scaled frequencies.
        dict(name="rotary_long", op="rotary", b=4, h=16, s=8192, d=128, rot=64,
             layout="interleaved", dtype="bfloat16", backward=False, fused=False, start=500000,
             factor=8.0),
        # One decoding step of 64 sequences with shared key heads, a 16-bit cache.
        dict(name="append_token", op="append", b=64, h=32, hk=8, s=1, d=128, rot=128,
             layout="half", dtype="bfloat16", cache="bfloat16", page=16, order="head", lo=1,
             hi=2048, ragged=False, factor=1.0),
        # A batch of prompts of unequal lengths, fp32 activations into a 16-bit cache.
        dict(name="append_prompt", op="append", b=8, h=16, hk=16, s=1500, d=64, rot=64,
             layout="half", dtype="float32", cache="bfloat16", page=64, order="token", lo=1500,
             hi=3500, ragged=True, factor=1.0),
        # One short sequence: the least a decoding step can cost.
        dict(name="attend_short", op="attend", b=1, h=6, hk=6, s=1, d=64, dtype="float32",
             cache="float32", page=16, order="token", lo=240, hi=240),
        # A serving batch of unequal lengths, four query heads to a key head.
        dict(name="attend_batch", op="attend", b=64, h=32, hk=8, s=1, d=128, dtype="bfloat16",
             cache="bfloat16", page=16, order="head", lo=1, hi=8192),
        # Two very long contexts: fp32 queries over a 16-bit cache.
        dict(name="attend_long", op="attend", b=2, h=16, hk=4, s=1, d=64, dtype="float32",
             cache="bfloat16", page=64, order="token", lo=131071, hi=131071),
        # fp32 throughout, a key head to each query head.
        dict(name="attend_f32", op="attend", b=16, h=16, hk=16, s=1, d=64, dtype="float32",
             cache="float32", page=32, order="token", lo=1000, hi=6000),
        # One new token a sequence over a short encoding (the canvas batch).
        dict(name="cross_token", op="cross", b=64, h=6, hk=6, sq=1, sk=240, d=64, lo=200, hi=240,
             backward=False),
        # A training step at the canvas batch: a padded batch of longer encodings.
        dict(name="cross_train", op="cross", b=64, h=6, hk=6, sq=240, sk=600, d=64, lo=100,
             hi=600, backward=True),
        # A training step with shared key heads over a long encoding.
        dict(name="cross_long", op="cross", b=4, h=16, hk=4, sq=2048, sk=8192, d=64, lo=8192,
             hi=8192, backward=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "cross", "cross"])
    d = rng.choice([32, 64, 64, 128])
    types = [("float32", "float32"), ("float32", "bfloat16"), ("float32", "float16"),
             ("bfloat16", "bfloat16"), ("float16", "float16")]
    dtype, cache = rng.choice(types)
    layout = rng.choice(["half", "interleaved"])
    hk, group = rng.choice([1, 2, 3, 4, 6, 8, 16]), rng.choice([1, 1, 2, 3, 4, 8])
    order, page = rng.choice(["token", "head"]), rng.choice([1, 8, 16, 24, 32, 64, 128, 256])
    if op == "rotary":
        d = rng.choice([32, 40, 64, 80, 128, 256])
        b, h = _log(rng, 1, 64), rng.randint(1, 32)
        s = max(1, min(_log(rng, 1, 16384), 60_000_000 // (b * h * d)))
        rot = rng.choice([d, d, d // 2, 2 * rng.randint(1, d // 2)])
        return dict(op=op, b=b, h=h, s=s, d=d, rot=rot, layout=layout, dtype=dtype,
                    backward=rng.random() < 0.5, fused=rng.random() < 0.5,
                    start=_log(rng, 1, 1_000_000) - 1, factor=rng.choice([1.0, 4.0, 32.0]))
    if op == "append":
        b, s = _log(rng, 1, 64), _log(rng, 1, 2048)
        s = max(1, min(s, 20_000_000 // (b * hk * (group + 2) * d)))
        lo = s + rng.randint(0, 500)
        return dict(op=op, b=b, h=hk * group, hk=hk, s=s, d=d, rot=rng.choice([d, d // 2]),
                    layout=layout, dtype=dtype, cache=cache, page=page, order=order, lo=lo,
                    hi=lo + rng.randint(0, 1000), ragged=rng.random() < 0.5,
                    factor=rng.choice([1.0, 4.0]))
    if op == "attend":
        b = _log(rng, 1, 128)
        hi = max(8, min(_log(rng, 8, 131072), 100_000_000 // (b * hk * d)))
        return dict(op=op, b=b, h=hk * group, hk=hk, s=rng.choice([1, 1, 1, 1, 2, 5]), d=d,
                    dtype=dtype, cache=cache, page=page, order=order,
                    lo=rng.choice([0, hi // 2, hi]), hi=hi)
    b, sq, sk = _log(rng, 1, 64), _log(rng, 1, 2048), _log(rng, 1, 8192)
    cap = 200_000_000 // (b * hk * group)  # the plain form holds every score
    while sq * sk > cap:
        sq, sk = max(1, sq * 3 // 4), max(1, sk * 3 // 4)
    sq = min(sq, max(1, 20_000_000 // (b * hk * group * d)))
    sk = min(sk, max(1, 20_000_000 // (b * hk * d)))
    return dict(op=op, b=b, h=hk * group, hk=hk, sq=sq, sk=sk, d=d,
                lo=rng.choice([0, sk // 2, sk]), hi=sk, backward=rng.random() < 0.6)


def _lengths(case):
    """The sequences' lengths: spread over lo .. hi, hi among them, by the case alone."""
    r = random.Random(case["b"] * 1_000_003 + case["hi"] * 1009 + case["lo"])
    return [case["hi"]] + [r.randint(case["lo"], case["hi"]) for _ in range(case["b"] - 1)]


def _new_tokens(case):
    """How many of the s new tokens each sequence has (all of them, or in a padded batch fewer)."""
    if not case.get("ragged"):
        return [case["s"]] * case["b"]
    r = random.Random(case["b"] * 7919 + case["s"])
    return [case["s"]] + [r.randint(0, case["s"]) for _ in range(case["b"] - 1)]


def _size(name):
    return {"float32": 4, "float16": 2, "bfloat16": 2}[name]


def work(case):
    b, d = case["b"], case["d"]
    if case["op"] == "rotary":
        n = b * case["h"] * case["s"] * d
        passes = 2 if case["backward"] else 1
        pairs = b * case["h"] * case["s"] * case["rot"] // 2
        return {"bytes": passes * 2 * n * _size(case["dtype"]), "flops": passes * 6 * pairs}
    if case["op"] == "append":
        n = sum(_new_tokens(case))
        e, c = _size(case["dtype"]), _size(case["cache"])
        h, hk = case["h"], case["hk"]
        # q is read and written whole: its padded rows come back as well
        moved = 2 * b * case["s"] * h * d * e + n * 2 * hk * d * (e + c)
        return {"bytes": moved, "flops": 6 * n * (h + hk) * case["rot"] // 2}
    if case["op"] == "attend":
        n = sum(_lengths(case))
        e, c = _size(case["dtype"]), _size(case["cache"])
        return {"bytes": 2 * n * case["hk"] * d * c + 2 * b * case["h"] * case["s"] * d * e,
                "flops": 4 * n * case["h"] * case["s"] * d}
    n = sum(_lengths(case))
    q, kv = b * case["h"] * case["sq"] * d, n * case["hk"] * d
    pairs = n * case["h"] * case["sq"]
    if not case["backward"]:
        return {"bytes": 4 * (2 * q + 2 * kv), "flops": 4 * pairs * d}
    # forward: q, k, v in, o out; backward: dO in, dq, dk, dv out (the whole of the padded dk, dv)
    pad = b * case["sk"] * case["hk"] * d
    return {"bytes": 4 * (4 * q + 2 * kv + 2 * pad), "flops": 14 * pairs * d}


def _frequencies(rot, factor, device):
    """Radians a position, 64 bits: base 10000, divided by `factor`, and the amplitude."""
    j = torch.arange(rot // 2, dtype=torch.float64, device=device)
    return 10000.0 ** (-2.0 * j / rot) / factor, 0.1 * math.log(factor) + 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dtype="float32"):
        x = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32)
        return x.to(getattr(torch, dtype))

    st = dict(case=case)
    b, d = case["b"], case["d"]
    if case["op"] == "rotary":
        h, s = case["h"], case["s"]
        x = normal(b, s, 3 if case["fused"] else 1, h, d, dtype=case["dtype"])
        st["x"] = x[:, :, 0].transpose(1, 2).requires_grad_(case["backward"])
        st["dy"] = normal(b, h, s, d, dtype=case["dtype"]) if case["backward"] else None
        start = torch.randint(0, 100, (b, 1), generator=gen, device=dev) + case["start"]
        st["positions"] = start + torch.arange(s, device=dev)
        st["freqs"], st["amplitude"] = _frequencies(case["rot"], case["factor"], dev)
        return st
    if case["op"] == "cross":
        st["q"] = normal(b, case["sq"], case["h"], d).transpose(1, 2)
        kv = normal(b, case["sk"], 2, case["hk"], d)
        st["k"], st["v"] = kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)
        st["dout"] = normal(b, case["h"], case["sq"], d) if case["backward"] else None
        if case["backward"]:
            for name in ("q", "k", "v"):
                st[name].requires_grad_(True)
        st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
        st["scale"] = 1.0 / math.sqrt(d)
        return st
    page, hk, lens = case["page"], case["hk"], _lengths(case)
    used = [-(-n // page) for n in lens]
    width, pages = max(max(used), 1), sum(used) + 3
    order = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32)
    host, at = order.cpu(), 0
    for i, n in enumerate(used):
        table[i, :n] = host[at:at + n]
        at += n
    st["table"] = table.to(dev)
    st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    shape = (pages, page, hk, d) if case["order"] == "token" else (pages, hk, page, d)
    for name in ("k_cache", "v_cache"):
        c = normal(*shape, dtype=case["cache"])
        st[name] = c if case["order"] == "token" else c.transpose(1, 2)
    qkv = normal(b, case["s"], case["h"] + 2 * hk, d, dtype=case["dtype"]).transpose(1, 2)
    st["q"] = qkv[:, :case["h"]]
    if case["op"] == "append":
        st["k"], st["v"] = qkv[:, case["h"]:-hk], qkv[:, -hk:]
        st["new"] = torch.tensor(_new_tokens(case), dtype=torch.int32, device=dev)
        st["freqs"], st["amplitude"] = _frequencies(case["rot"], case["factor"], dev)
    else:
        st["scale"] = 1.0 / math.sqrt(d)
    return st


# --- the plain forms --------------------------------------------------------------------------


def _rotate(x, positions, freqs, amplitude, interleaved, inverse=False):
    """x [b, h, s, d] rotated at positions [b, s]: fp32, the angles in 64 bits."""
    angle = positions.double()[:, None, :, None] * freqs
    c, s = (amplitude * angle.cos()).float(), (amplitude * angle.sin()).float()
    if inverse:
        s = -s
    r = 2 * freqs.numel()
    y = x.float().clone()
    if interleaved:
        a, z = x[..., 0:r:2].float(), x[..., 1:r:2].float()
        y[..., 0:r:2], y[..., 1:r:2] = a * c - z * s, z * c + a * s
    else:
        a, z = x[..., :r // 2].float(), x[..., r // 2:r].float()
        y[..., :r // 2], y[..., r // 2:r] = a * c - z * s, z * c + a * s
    return y


def _probabilities(scores, allowed):
    """Softmax over the allowed keys; a row without any is zero."""
    scores = scores.masked_fill(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).min)
    p = (scores - top).exp()
    return p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(scores.dtype).tiny)


def _cross_plain(st):
    q, k, v, scale = st["q"], st["k"], st["v"], st["scale"]
    (b, h, sq, d), (hk, sk) = q.shape, k.shape[1:3]
    qg = q.reshape(b, hk, -1, d)  # the heads of a group beside each other
    allowed = torch.arange(sk, device=q.device) < st["lengths"][:, None, None, None]
    p = _probabilities(torch.matmul(qg, k.transpose(2, 3)) * scale, allowed)
    out = torch.matmul(p, v)
    if st["dout"] is None:
        return out.reshape(b, h, sq, d)
    g = st["dout"].reshape(b, hk, -1, d)
    dv = torch.matmul(p.transpose(2, 3), g)
    ds = p * (torch.matmul(g, v.transpose(2, 3)) - (g * out).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k).reshape(b, h, sq, d)
    return out.reshape(b, h, sq, d), dq, torch.matmul(ds.transpose(2, 3), qg), dv


def _slots(st, positions):
    """(page, row in the page) of logical positions [b, n]."""
    page = st["case"]["page"]
    at = (positions // page).clamp(0, st["table"].shape[1] - 1)
    return st["table"].long().gather(1, at), positions % page


def _append_plain(st):
    case, q, k, v = st["case"], st["q"], st["k"], st["v"]
    i = torch.arange(case["s"], device=q.device)
    valid = i < st["new"][:, None]
    positions = (st["lengths"] - st["new"]).long()[:, None] + i
    inter = case["layout"] == "interleaved"
    turn = [_rotate(x, positions, st["freqs"], st["amplitude"], inter) for x in (q, k)]
    pages, rows = (x[valid] for x in _slots(st, torch.where(valid, positions, 0)))
    st["k_cache"][pages, rows] = turn[1].transpose(1, 2)[valid].to(st["k_cache"].dtype)
    st["v_cache"][pages, rows] = v.transpose(1, 2)[valid].to(st["v_cache"].dtype)
    # rows behind a sequence's last new token come back as zeros
    out = torch.where(valid[:, None, :, None], turn[0], 0.0).to(q.dtype)
    return out, st["k_cache"], st["v_cache"]


def _attend_plain(st):
    case, q = st["case"], st["q"]
    (b, h, s, d), hk = q.shape, case["hk"]
    n = max(1, case["hi"])
    j = torch.arange(n, device=q.device)
    pages, rows = _slots(st, j.expand(b, n))
    pages = pages.clamp_min(0)
    k = st["k_cache"][pages, rows].transpose(1, 2).float()
    v = st["v_cache"][pages, rows].transpose(1, 2).float()
    # new token i sees the keys up to its own
    limit = st["lengths"][:, None] - s + 1 + torch.arange(s, device=q.device)
    allowed = (j < limit[:, :, None])[:, None].expand(b, h // hk, s, n).reshape(b, 1, -1, n)
    qg = q.float().reshape(b, hk, -1, d)
    p = _probabilities(torch.matmul(qg, k.transpose(2, 3)) * st["scale"], allowed)
    return torch.matmul(p, v).reshape(b, h, s, d).to(q.dtype)


def run(state):
    case = state["case"]
    inter = case.get("layout") == "interleaved"
    if own:
        cfa = _cfa()
        if case["op"] == "rotary":
            y = cfa.rotary(state["x"], state["positions"], state["freqs"],
                           amplitude=state["amplitude"], interleaved=inter)
            if not case["backward"]:
                return y
            return y, torch.autograd.grad(y, state["x"], state["dy"])[0]
        if case["op"] == "cross":
            qkv = state["q"], state["k"], state["v"]
            out = cfa.cross_attention(*qkv, state["scale"], key_lengths=state["lengths"])
            if not case["backward"]:
                return out
            return out, *torch.autograd.grad(out, qkv, state["dout"])
        if case["op"] == "append":
            q = cfa.paged_append(state["k"], state["v"], state["k_cache"], state["v_cache"],
                                 state["table"], state["lengths"], q=state["q"],
                                 freqs=state["freqs"], amplitude=state["amplitude"],
                                 interleaved=inter, new_lengths=state["new"])
            return q, state["k_cache"], state["v_cache"]
        return cfa.paged_attention(state["q"], state["k_cache"], state["v_cache"],
                                   state["table"], state["lengths"], state["scale"])
    with torch.no_grad():
        if case["op"] == "rotary":
            rest = state["positions"], state["freqs"], state["amplitude"], inter
            y = _rotate(state["x"], *rest).to(state["x"].dtype)
            if not case["backward"]:
                return y
            return y, _rotate(state["dy"], *rest, inverse=True).to(state["x"].dtype)
        if case["op"] == "cross":
            return _cross_plain(state)
        return _append_plain(state) if case["op"] == "append" else _attend_plain(state)


# --- the definitions in 64 bits ---------------------------------------------------------------


def _turned(x, positions, freqs, amplitude, interleaved, sign):
    """Each pair as a complex number times amplitude e^{i sign angle}."""
    half = freqs.numel()
    x = x.detach().double()
    if interleaved:
        z = torch.view_as_complex(x[..., :2 * half].unflatten(-1, (half, 2)).contiguous())
    else:
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous())
    angle = sign * torch.einsum("bs,j->bsj", positions.double(), freqs)[:, None]
    z = z * torch.polar(torch.full_like(angle, amplitude), angle)
    parts = torch.view_as_real(z)
    flat = parts.flatten(-2) if interleaved else torch.cat((parts[..., 0], parts[..., 1]), -1)
    return torch.cat((flat, x[..., 2 * half:]), -1)


def _attended(q, k, v, scale, counts):
    """One key head: q [n, d] over the first counts[r] keys each, in 64 bits -> (p, o)."""
    score = torch.einsum("nd,kd->nk", q, k) * scale
    seen = torch.arange(k.shape[0], device=q.device)[None] < counts[:, None]
    weight = torch.where(seen, torch.exp(score - torch.where(
        seen, score, -1e300).max(1, keepdim=True).values), torch.zeros_like(score))
    total = weight.sum(1, keepdim=True)
    p = torch.where(total > 0, weight / torch.where(total > 0, total, torch.ones_like(total)),
                    torch.zeros_like(weight))
    return p, p @ v


def exact(case, seed):
    st = prepare(case, seed)
    inter = case.get("layout") == "interleaved"
    if case["op"] == "rotary":
        rest = st["positions"], st["freqs"], st["amplitude"], inter
        y = _turned(st["x"], *rest, 1.0)
        return (y, _turned(st["dy"], *rest, -1.0)) if case["backward"] else y
    if case["op"] == "append":
        caches = [st["k_cache"].double(), st["v_cache"].double()]
        out = torch.zeros(st["q"].shape, dtype=torch.float64, device=st["q"].device)
        for i, (n, new) in enumerate(zip(_lengths(case), _new_tokens(case))):
            if new == 0:
                continue
            at = torch.arange(n - new, n, device=out.device)
            rest = at[None], st["freqs"], st["amplitude"], inter, 1.0
            out[i, :, :new] = _turned(st["q"][i:i + 1, :, :new], *rest)[0]
            page, row = st["table"][i].long()[at // case["page"]], at % case["page"]
            caches[0][page, row] = _turned(st["k"][i:i + 1, :, :new], *rest)[0].transpose(0, 1)
            caches[1][page, row] = st["v"][i, :, :new].double().transpose(0, 1)
        return out, *caches
    q = st["q"].detach().double()
    group = case["h"] // case["hk"]
    if case["op"] == "attend":
        out, s = torch.zeros_like(q), case["s"]
        for i, n in enumerate(_lengths(case)):
            if n == 0:
                continue
            at = torch.arange(n, device=q.device)
            page, row = st["table"][i].long()[at // case["page"]], at % case["page"]
            k, v = st["k_cache"][page, row].double(), st["v_cache"][page, row].double()
            counts = (n - s + 1 + torch.arange(s, device=q.device)).repeat(group)
            for j in range(case["hk"]):
                rows = q[i, j * group:(j + 1) * group].reshape(-1, case["d"])
                o = _attended(rows, k[:, j], v[:, j], st["scale"], counts)[1]
                out[i, j * group:(j + 1) * group] = o.view(group, s, -1)
        return out
    k, v = st["k"].detach().double(), st["v"].detach().double()
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    for i, n in enumerate(_lengths(case)):
        for j in range(case["hk"]):
            heads = slice(j * group, (j + 1) * group)
            rows = q[i, heads].reshape(-1, case["d"])
            counts = torch.full((rows.shape[0],), n, device=q.device)
            p, o = _attended(rows, k[i, j], v[i, j], st["scale"], counts)
            out[i, heads] = o.view(group, -1, case["d"])
            if case["backward"]:
                g = st["dout"][i, heads].double().reshape(-1, case["d"])
                dp = g @ v[i, j].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * st["scale"]
                dq[i, heads] = (ds @ k[i, j]).view(group, -1, case["d"])
                dk[i, j], dv[i, j] = ds.T @ rows, p.T @ g
    return (out, dq, dk, dv) if case["backward"] else out

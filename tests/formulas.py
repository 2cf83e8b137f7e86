# SPDX-License-Identifier: MIT OR Apache-2.0
"""Test helper: the operators beside the fused attention in 64 bits, straight from their formulas, on
the CPU."""

from __future__ import annotations

import torch


def rotate(x, positions, freqs, amplitude=1.0, interleaved=False, inverse=False):
    """x [b, h, s, d] -> float64; positions [s] or [b, s], freqs float64 [r / 2]."""
    x = x.detach().cpu().double().clone()
    positions, freqs = positions.cpu().double(), freqs.cpu()
    positions = positions.expand(x.shape[0], x.shape[2])
    angle = positions[:, None, :, None] * freqs
    c, s = amplitude * angle.cos(), amplitude * angle.sin() * (-1.0 if inverse else 1.0)
    r = 2 * freqs.numel()
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, z = x[..., one].clone(), x[..., two].clone()
    x[..., one], x[..., two] = a * c - z * s, z * c + a * s
    return x


def rotate_band(x, freqs, amplitude=1.0, interleaved=False, dtype=torch.float32):
    """How far a rotation may be off, per element: with u = 2^-24, the angle's last rounding is half
    a step of at most 1/2 turn (2 pi 2^-26 radians = 1.6 u), sincospi is off by 2 steps (4 u at
    most), cos and sin are scaled once (u), the product and the fused sum round once each (2 u) of at
    most A (|x1| + |x2|): 8.6 u, then half a step of the output's type."""
    x = x.detach().cpu().double().abs()
    r = 2 * freqs.numel()
    size = torch.zeros_like(x)
    one, two = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    size[..., one] = size[..., two] = abs(amplitude) * (x[..., one] + x[..., two])
    band = 8.6 * 2.0 ** -24 * size
    if dtype != torch.float32:
        full = torch.where(size > 0, size, x)
        tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0  # half the smallest fp16 step
        band = band + torch.finfo(dtype).eps / 2 * full + tiny
    return band


def attend(q, k, v, scale, seen):
    """q [h, s, d], k and v [hk, n, d] (float64), seen [s] keys each -> o [h, s, d]."""
    h, s, d = q.shape
    group = h // k.shape[0]
    out = torch.zeros_like(q)
    for i in range(h):
        for j in range(s):
            n = int(seen[j])
            if n <= 0:
                continue
            y = (k[i // group, :n] @ q[i, j]) * scale
            p = torch.softmax(y, 0)
            out[i, j] = p @ v[i // group, :n]
    return out


def cross(q, k, v, scale, lengths, dout=None):
    """q [b, h, sq, d], k and v [b, hk, sk, d] -> o, and with dout dq, dk, dv, in float64; and the same
    with every product and difference taken of absolute values (what roundings are relative to)."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    b, h, sq, d = q.shape
    hk, sk = k.shape[1:3]
    group = h // hk if hk else 1
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    ao, aq, ak, av = (torch.zeros_like(t) for t in (q, q, k, v))
    for i in range(b):
        n = sk if lengths is None else max(0, min(sk, int(lengths[i])))
        if n == 0:
            continue
        for j in range(h):
            kj, vj = k[i, j // group, :n], v[i, j // group, :n]
            p = torch.softmax(q[i, j] @ kj.T * scale, -1)
            o[i, j] = p @ vj
            ao[i, j] = p @ vj.abs()
            if dout is not None:
                g = dout[i, j].detach().cpu().double()
                ds = p * (g @ vj.T - (g * o[i, j]).sum(-1, keepdim=True)) * scale
                dq[i, j] = ds @ kj
                dk[i, j // group, :n] += ds.T @ q[i, j]
                dv[i, j // group, :n] += p.T @ g
                size = p * (g.abs() @ vj.T.abs() + (g.abs() * ao[i, j]).sum(-1, keepdim=True)) * abs(scale)
                aq[i, j] = size @ kj.abs()
                ak[i, j // group, :n] += size.T @ q[i, j].abs()
                av[i, j // group, :n] += p.T @ g.abs()
    return (o, ao) if dout is None else ((o, dq, dk, dv), (ao, aq, ak, av))


def paged(k, v, page, gen, dtype, spare=2, order="token", fill=float("nan")):
    """Lists of float tensors [hk, n_b, d] as a cache of `page`-row pages in shuffled order, unused
    rows holding `fill`: (k_cache, v_cache, page_table, lengths), on the CPU."""
    hk, d = k[0].shape[0], k[0].shape[2]
    used = [-(-x.shape[1] // page) for x in k]
    pages = sum(used) + spare
    shape = (pages, page, hk, d) if order == "token" else (pages, hk, page, d)
    caches = [torch.full(shape, fill, dtype=dtype) for _ in range(2)]
    views = [c if order == "token" else c.transpose(1, 2) for c in caches]
    perm = torch.randperm(pages, generator=gen)
    table = torch.full((len(k), max(max(used), 1)), -7, dtype=torch.int32)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = perm[at:at + n].int()
        at += n
        for c, src in zip(views, (k[i], v[i])):
            for r in range(src.shape[1]):
                c[table[i, r // page], r % page] = src[:, r].to(dtype)
    return views[0], views[1], table, torch.tensor([x.shape[1] for x in k], dtype=torch.int32)

# SPDX-License-Identifier: MIT OR Apache-2.0
"""What autograd may not ask of the operators is refused, on the CPU (before a device is looked at)."""

import pytest
import torch
from torch.autograd import forward_ad

import candle_fused_attn as cfa


def operands():
    q, k = torch.zeros(2, 4, 1, 64), torch.zeros(2, 2, 1, 64)
    pool = torch.zeros(3, 16, 2, 64)
    table, lengths = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    return dict(q=q, k=k, v=k.clone(), kc=pool, vc=pool.clone(), table=table, lengths=lengths,
                freqs=torch.ones(32, dtype=torch.float64), qkv=torch.zeros(2, 1, 192))


CALLS = {
    "cross_attention": (lambda a: cfa.cross_attention(a["q"], a["k"], a["v"], 0.1), "q k v"),
    "rotary": (lambda a: cfa.rotary(a["q"], 0, a["freqs"]), "q freqs"),
    "rotary_qkv": (lambda a: cfa.rotary_qkv(a["qkv"], 1, 0, a["freqs"]), "qkv freqs"),
    "paged_append": (lambda a: cfa.paged_append(a["k"], a["v"], a["kc"], a["vc"], a["table"],
                                                a["lengths"], q=a["q"], freqs=a["freqs"]),
                     "q k v kc vc freqs"),
    "paged_attention": (lambda a: cfa.paged_attention(a["q"], a["kc"], a["vc"], a["table"],
                                                      a["lengths"], 0.1), "q kc vc"),
}


@pytest.mark.parametrize("name,which", [(n, w) for n, (_, ws) in CALLS.items() for w in ws.split()])
def test_forward_mode_tangents_are_refused(name, which):
    """A dual tensor has no requires_grad; a result without its tangent would read as a derivative of zero."""
    call, a = CALLS[name][0], operands()
    for no_grad in (False, True):  # (forward mode does not look at it)
        with forward_ad.dual_level(), torch.set_grad_enabled(not no_grad):
            dual = {**a, which: forward_ad.make_dual(a[which], torch.ones_like(a[which]))}
            with pytest.raises(cfa.FusedAttentionError, match="no forward-mode derivative"):
                call(dual)
    with pytest.raises(cfa.FusedAttentionError, match="CUDA"):
        call(a)

# SPDX-License-Identifier: MIT OR Apache-2.0
"""The operators beside the fused attention as a compiled extension (_ops.so, from
binding/torch_ops.cpp), bound to the library that `_abi` loads, to this package's error and to its
failure detection. Loading fails loudly when either library is missing."""

from __future__ import annotations

import ctypes

from . import FusedAttentionError, _abi, _raise_if_expired, _sink_flag

try:
    from . import _ops
except ImportError as e:
    raise ImportError(
        "candle_fused_attn: _ops.so is missing or does not fit this torch; build it with "
        f"`python __graft_entry__.py build` ({e})") from e

# In the order of the extension's table.
_ENTRY_POINTS = (
    "cfa_cross_fwd_f32", "cfa_cross_bwd_workspace_bytes_fast", "cfa_cross_bwd_f32",
    "cfa_cross_few_workspace_bytes", "cfa_cross_few_f32", "cfa_rotary", "cfa_paged_append",
    "cfa_paged_attention_workspace_bytes", "cfa_paged_attention", "cfa_strerror")

_lib = _abi.load()
_ops.bind(tuple(ctypes.cast(getattr(_lib, name), ctypes.c_void_p).value for name in _ENTRY_POINTS),
          FusedAttentionError, lambda: ctypes.addressof(_sink_flag()), _raise_if_expired)


def require(ok: bool, who: str, what: str) -> None:
    if not ok:
        raise FusedAttentionError(f"{who}: {what}")

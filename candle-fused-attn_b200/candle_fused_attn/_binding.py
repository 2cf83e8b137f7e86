# SPDX-License-Identifier: MIT OR Apache-2.0
"""The operators beside the fused attention as a compiled extension (_ops.so, from
binding/torch_ops.cpp), bound to the library that `_abi` loads, to this package's error and to its
failure detection. Both are loaded when one of these operators is first called: the fused attention
needs nothing of the extension, which fits only the torch it was built against."""

from __future__ import annotations

import ctypes
import threading

from . import FusedAttentionError, _abi, _raise_if_expired, _sink_flag

# In the order of the extension's table.
_ENTRY_POINTS = (
    "cfa_cross_fwd_f32", "cfa_cross_bwd_workspace_bytes", "cfa_cross_bwd_workspace_bytes_fast",
    "cfa_cross_bwd_f32", "cfa_cross_few_workspace_bytes", "cfa_cross_few_f32", "cfa_rotary", "cfa_paged_append",
    "cfa_paged_attention_workspace_bytes", "cfa_paged_attention", "cfa_strerror")
_FUNCTIONS = ("cross_attention", "paged_append", "paged_attention", "rotary", "rotary_qkv")


class _Ops:
    """The extension's functions as attributes; the first one asked for loads it (loudly, when either
    library is missing) and leaves them all here."""

    _lock = threading.Lock()

    def __getattr__(self, name: str):
        if name not in _FUNCTIONS:
            raise AttributeError(name)
        with self._lock:
            if name not in self.__dict__:
                self._load()
        return self.__dict__[name]

    def _load(self) -> None:
        try:
            from . import _ops as ext
        except ImportError as e:
            raise ImportError(
                "candle_fused_attn: _ops.so is missing or does not fit this torch; build it with "
                f"`python __graft_entry__.py build` ({e})") from e
        lib = _abi.load()
        ext.bind(tuple(ctypes.cast(getattr(lib, entry), ctypes.c_void_p).value for entry in _ENTRY_POINTS),
                 FusedAttentionError, lambda: ctypes.addressof(_sink_flag()), _raise_if_expired)
        self.__dict__.update((f, getattr(ext, f)) for f in _FUNCTIONS)


_ops = _Ops()


def require(ok: bool, who: str, what: str) -> None:
    if not ok:
        raise FusedAttentionError(f"{who}: {what}")

# SPDX-License-Identifier: MIT OR Apache-2.0
"""Importing the package loads no native library; the operators' extension is loaded by the first call of
one of them, and without it the rest works."""

import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "candle-fused-attn_b200"


def python(code):
    head = f"import sys; sys.path.insert(0, {str(PACKAGE)!r})\n"
    r = subprocess.run([sys.executable, "-c", head + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_import_loads_no_library():
    out = python("""
import torch, candle_fused_attn as cfa
maps = lambda: open("/proc/self/maps").read()
assert "candle_fused_attn._ops" not in sys.modules
assert "_ops.so" not in maps() and "libcfa.so" not in maps()
f, _ = cfa.rotary_frequencies(8, device="cpu")
assert "_ops.so" not in maps()
try:
    cfa.rotary(torch.zeros(1, 1, 2, 8), 0, f)
except cfa.FusedAttentionError as e:
    print(e)
assert "_ops.so" in maps() and "libcfa.so" in maps()
""")
    assert "CUDA tensors required" in out


def test_without_the_extension():
    """None in its place, as an extension built against another torch raises ImportError."""
    out = python("""
sys.modules["candle_fused_attn._ops"] = None
import torch, candle_fused_attn as cfa
x = torch.zeros(1, 1, 2, 64)
try:
    cfa.fused_attention(x, x, x, 0.125, False)
except cfa.FusedAttentionError as e:
    print("fused:", e)
for _ in range(2):
    try:
        cfa.cross_attention(x, x, x, 0.125)
    except ImportError as e:
        print("cross:", e)
del sys.modules["candle_fused_attn._ops"]  # (built since)
try:
    cfa.cross_attention(x, x, x, 0.125)
except cfa.FusedAttentionError as e:
    print("then:", e)
""")
    assert "fused: fused_attention: CUDA tensors required" in out
    assert out.count("_ops.so is missing or does not fit this torch") == 2
    assert "then: cross_attention: CUDA tensors required" in out


def test_threads_load_it_once():
    out = python("""
import threading, torch, candle_fused_attn as cfa
x, start, seen = torch.zeros(1, 1, 2, 64), threading.Barrier(8), []
def call():
    start.wait()
    try:
        cfa.cross_attention(x, x, x, 0.125)
    except Exception as e:
        seen.append(type(e).__name__)
ts = [threading.Thread(target=call) for _ in range(8)]
[t.start() for t in ts]
[t.join() for t in ts]
print(seen)
""")
    assert out.count("FusedAttentionError") == 8


def test_the_extension_has_no_cxx_runtime_of_its_own():
    """It throws what torch catches: one libstdc++ in the process, none inside the extension."""
    readelf = shutil.which("readelf")
    if readelf is None:
        pytest.skip("no readelf")
    lib = str(PACKAGE / "candle_fused_attn" / "_ops.so")
    needed = subprocess.run([readelf, "-dW", lib], capture_output=True, text=True, check=True).stdout
    assert "[libstdc++.so.6]" in needed
    names = subprocess.run([readelf, "--dyn-syms", "-W", lib], capture_output=True, text=True, check=True).stdout
    own = [x.split()[-1] for x in names.splitlines() if "__cxa_throw" in x or "_ZNSt6locale" in x]
    assert own and all(" UND " in x for x in names.splitlines() if "__cxa_throw" in x or "_ZNSt6locale" in x), own

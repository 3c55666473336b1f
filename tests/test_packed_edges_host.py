"""The packed operators' host sides at the ends of their ranges; no GPU needed: every call is answered or refused before
a launch."""

import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from modelopt_amd import _ext

ROOT = Path(__file__).resolve().parents[1]


def test_attention_workspace_of_any_bound():
    """Row counts past 32 bits: no size, no end of the process (a count of tiles that wraps to 0 divides)."""
    code = f"""
import ctypes
lib = ctypes.CDLL({str(_ext.KERNEL_LIB)!r})
f = lib.mtq_kv_attention_workspace_bytes
f.argtypes, f.restype = [ctypes.c_int] * 6, ctypes.c_size_t
for batch, heads, kv, d, lq, lk in ((1, 1 << 20, 1, 256, 1 << 16, 4096), (1, 1 << 20, 1, 128, 1 << 20, 4096),
                                    (3, 32, 1, 256, 2 ** 31 - 1, 4096), (65535, 8, 8, 64, 2 ** 31 - 1, 0), (1, 4, 4, 64, 1, -5)):
    assert f(batch, heads, kv, d, lq, lk) == 0, (heads, d, lq)
print("answered")
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and "answered" in run.stdout, (run.returncode, run.stderr)

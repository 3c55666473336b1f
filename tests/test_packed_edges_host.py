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


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would launch")
def test_attention_is_not_refused_the_workspace_that_it_asked_for():
    """Bounds of the keys above the table's positions, for which fewer keys mean a larger workspace."""
    from test_packed_ops_host import ARG, FAKE, I64, BF16, kv_cache

    lib = _ext.kernel_cdll()
    size, attend = lib.mtq_kv_attention_workspace_bytes, lib.mtq_kv_attention
    P, I, F64, SZ = ctypes.c_void_p, ctypes.c_int, ctypes.c_double, ctypes.c_size_t
    size.argtypes, size.restype = [I] * 6, SZ
    attend.argtypes = [P, P, P, P, I64, I, P, I64, I, P, P, P, I, I, I, I, F64, I, P, SZ, P]
    strides = (I64 * 4)(4096, 128, 4096, 128)
    for batch in (1, 3, 38, 100):
        for lq in (1, 64):
            for lk in (0, 1, 600, 1500, 1537, 1600, 2500, 100000, 2 ** 31 - 1):
                need = size(batch, 32, 8, 128, lq, lk)
                status = attend(ctypes.byref(kv_cache(page_size=64)), FAKE, FAKE, strides, batch * lq, 32, FAKE, 24, 24, FAKE, FAKE, FAKE,
                                batch, lq, lk, 1, 0.1, BF16, FAKE, need, None)
                assert status != ARG, (batch, lq, lk, need)


def test_what_an_op_writes_is_declared():
    """A graph pass may drop or move a call whose schema says that it changes nothing."""
    _ext.require_ops()
    ops = torch.ops.modelopt_amd
    for name, written in (("kv_append", {"cache"}), ("kv_read", {"k", "v"}), ("kv_attention", {"o"})):
        schema = getattr(ops, name).default._schema
        assert schema.is_mutable, name
        assert {a.name for a in schema.arguments if a.alias_info is not None and a.alias_info.is_write} == written, name
    graph = torch.fx.Graph()
    x = graph.placeholder("x")
    graph.call_function(ops.kv_append.default, ([x] * 6, x, x, x, x, x, x, 1))
    graph.output(x)
    graph.eliminate_dead_code()
    assert any(n.target is ops.kv_append.default for n in graph.nodes)


def test_forward_mode_tangents_are_refused():
    """An operator without a derivative would drop them without a word."""
    from torch.autograd import forward_ad

    from modelopt_amd.torch.kernels.quantization.mx import refuse_grad

    x, w = torch.randn(4, 32), torch.zeros(4, dtype=torch.uint8)
    refuse_grad("op", x, w, None)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        refuse_grad("op", x, w, None)
        for no_grad in (False, True):
            with torch.set_grad_enabled(not no_grad), pytest.raises(NotImplementedError, match="forward only"):
                refuse_grad("op", w, d)
        refuse_grad("op", forward_ad.unpack_dual(d).primal)
    with pytest.raises(NotImplementedError, match="forward only"):
        torch.func.jvp(lambda t: refuse_grad("op", t), (x,), (x,))
    with pytest.raises(NotImplementedError, match="forward only"):
        torch.func.grad(lambda t: refuse_grad("op", t) or t.sum())(x)

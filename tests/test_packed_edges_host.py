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


def test_shapes_without_a_device():
    """The operators under FakeTensorMode: outputs' shapes and types, and the refusals that go by them."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from modelopt_amd.torch.kernels.common.attention import NVFP4KVCache
    from modelopt_amd.torch.kernels.quantization import mx_linear, mx_quantize, rms_norm_quantize

    _ext.require_ops()
    forms = {"mxfp4": (32, torch.uint8, (3, 5, 2), torch.uint8), "mxfp8": (64, torch.float8_e4m3fn, (3, 5, 2), torch.uint8),
             "fp8": (64, torch.float8_e4m3fn, (1,), torch.float32), "fp8_token": (64, torch.float8_e4m3fn, (3, 5, 1), torch.float32)}
    with FakeTensorMode():
        def new(*shape, dtype=torch.bfloat16):
            return torch.empty(*shape, dtype=dtype, device="cuda")

        x, w, ws = new(3, 5, 64), new(48, 32, dtype=torch.uint8), new(48, 2, dtype=torch.uint8)
        for fmt, (cols, qt, ss, st) in forms.items():
            amax = new(1, dtype=torch.float32) if fmt == "fp8" else None
            for q, s in (mx_quantize(x, fmt, amax), rms_norm_quantize(x, new(64), residual=x, format=fmt, amax=amax)[:2]):
                assert (*q.shape,) == (3, 5, cols) and q.dtype == qt and (*s.shape,) == ss and s.dtype == st
                y = mx_linear(q, w, ws, new(48), format=fmt, x_scale=s)
                assert (*y.shape,) == (3, 5, 48) and y.dtype == torch.bfloat16 and y.device.type == "cuda"
            assert mx_linear(x, w, ws, format=fmt, amax=amax, out_dtype=torch.float32).dtype == torch.float32
        assert rms_norm_quantize(x, new(64))[2] is None and rms_norm_quantize(x, new(64), residual=x)[2].shape == x.shape
        with pytest.raises(ValueError, match="multiple of 32"):
            mx_quantize(x[..., :40])
        with pytest.raises(ValueError, match="columns"):
            mx_linear(x, w[:, :16], ws[:, :1])
        cache = NVFP4KVCache(4, 16, 2, 64)
        n, table = new(1, dtype=torch.int32), new(1, 4, dtype=torch.int32)
        cache.append(new(7, 2, 64), new(7, 2, 64), n, n, n, table, 7)
        k, v = cache.read(n, n, n, table, 7, 9, dtype=torch.float16)
        assert (*k.shape,) == (*v.shape,) == (9, 2, 64) and k.dtype == torch.float16
        o = cache.attention(new(7, 8, 64), n, n, n, table, 7)
        assert (*o.shape,) == (7, 8, 64) and o.dtype == torch.bfloat16

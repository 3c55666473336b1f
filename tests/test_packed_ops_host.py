"""Refusals of the packed 4-bit operators (kernels.quantization, NVFP4KVCache) that need no GPU: the C entry
points check their arguments before any HIP call, the Python ones before they reach an op."""

import ctypes

import pytest
import torch

from modelopt_amd import _ext
from modelopt_amd.torch.kernels.common.attention import NVFP4KVCache
from modelopt_amd.torch.kernels.quantization import mx_linear, mx_quantize, rms_norm_quantize

P, I64, I, F64, SZ = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_double, ctypes.c_size_t
FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below is refused before
F32, F16, BF16, F64D = 0, 1, 2, 3
OK, ARG, DTYPE, FORMAT = 0, -1, -2, -4


class KvCache(ctypes.Structure):
    _fields_ = [("data", P * 2), ("scale", P * 2), ("data_strides", (I64 * 3) * 2), ("scale_strides", (I64 * 3) * 2),
                ("amax", P * 2), ("num_pages", I), ("page_size", I), ("num_kv_heads", I), ("head_dim", I)]


def kv_cache(**over):
    c = KvCache()
    for i in range(2):
        c.data[i] = c.scale[i] = c.amax[i] = 4096
        for j, n in enumerate((8 * 16 * 64, 16 * 64, 64)):
            c.data_strides[i][j] = n
            c.scale_strides[i][j] = n // 8
    c.num_pages, c.page_size, c.num_kv_heads, c.head_dim = 4, 16, 8, 128
    for k, v in over.items():
        setattr(c, k, v)
    return c


@pytest.fixture(scope="module")
def lib():
    lib = _ext.kernel_cdll()
    lib.mtq_mx_quantize.argtypes = [P, I64, I64, I64, I, I, P, P, P, P]
    lib.mtq_rms_norm_quantize.argtypes = [P, I64, P, I64, P, I, F64, P, P, P, P, I64, I64, I, I, P]
    lib.mtq_mx_linear.argtypes = [P, I64, I, P, I, P, P, P, P, I, P, I, I64, I64, I64, P, SZ, P]
    lib.mtq_mx_linear_workspace_bytes.argtypes = [I64, I64, I64, I, I]
    lib.mtq_mx_linear_workspace_bytes.restype = SZ
    lib.mtq_kv_append.argtypes = [P, P, P, P, I64, P, I64, I, P, P, P, I, I, I, P]
    lib.mtq_kv_attention.argtypes = [P, P, P, P, I64, I, P, I64, I, P, P, P, I, I, I, I, F64, I, P, SZ, P]
    lib.mtq_kv_attention_workspace_bytes.argtypes = [I, I, I, I, I, I]
    lib.mtq_kv_attention_workspace_bytes.restype = SZ
    return lib


def test_mx_quantize_refusals(lib):
    def call(x=FAKE, stride=64, rows=4, cols=64, dtype=BF16, kind=0, amax=None, q=FAKE, s=FAKE):
        return lib.mtq_mx_quantize(x, stride, rows, cols, dtype, kind, amax, q, s, None)

    assert call(kind=7) == FORMAT and call(kind=-1) == FORMAT
    assert call(dtype=F64D) == DTYPE
    assert call(cols=48) == ARG  # MX blocks of 32
    assert call(stride=32) == ARG  # rows that overlap
    assert call(x=None) == ARG and call(q=None) == ARG and call(s=None) == ARG
    assert call(kind=2) == ARG  # per tensor without amax
    assert call(q=ctypes.c_void_p(4097)) == ARG
    assert call(rows=0, x=None, q=None, s=None) == OK  # nothing to do
    assert call(rows=-1) == ARG and call(cols=0, kind=3) == ARG


def test_rms_norm_quantize_refusals(lib):
    def call(x=FAKE, w=FAKE, wd=BF16, eps=1e-6, r=None, h=None, q=FAKE, s=FAKE, amax=None, rows=4, cols=64, dtype=BF16, kind=1):
        return lib.mtq_rms_norm_quantize(x, cols, r, cols, w, wd, eps, h, q, s, amax, rows, cols, dtype, kind, None)

    assert call(kind=9) == FORMAT
    assert call(dtype=F64D) == DTYPE and call(wd=F16) == DTYPE
    assert call(cols=40) == ARG and call(cols=65536 + 32) == ARG
    assert call(eps=-1.0) == ARG and call(eps=float("nan")) == ARG
    assert call(r=FAKE) == ARG  # a residual needs somewhere to put the sum
    assert call(kind=2) == ARG and call(w=None) == ARG
    assert call(rows=0, x=None) == OK


def test_mx_linear_refusals(lib):
    def call(x=FAKE, stride=64, xd=BF16, xs=None, kind=0, amax=None, w=FAKE, ws=FAKE, bias=None, bd=BF16, y=FAKE, yd=BF16, m=20,
             n=16, k=64, wsp=FAKE, nb=1 << 30):
        return lib.mtq_mx_linear(x, stride, xd, xs, kind, amax, w, ws, bias, bd, y, yd, m, n, k, wsp, nb, None)

    assert call(kind=4) == FORMAT
    assert call(yd=F64D) == DTYPE and call(xd=F64D) == DTYPE and call(bias=FAKE, bd=F16) == DTYPE
    assert call(k=48) == ARG and call(n=0) == ARG and call(m=-1) == ARG and call(k=(1 << 22) + 32) == ARG
    assert call(w=ctypes.c_void_p(4100)) == ARG and call(ws=ctypes.c_void_p(4098)) == ARG
    assert call(xd=-1) == ARG  # quantised rows without their scales
    assert call(stride=32) == ARG and call(kind=2) == ARG
    assert call(wsp=None) == ARG and call(nb=16) == ARG  # rows by the workspace
    assert call(m=0, x=None, y=None) == OK
    assert lib.mtq_mx_linear_workspace_bytes(20, 16, 64, 0, BF16) > 0
    assert lib.mtq_mx_linear_workspace_bytes(0, 16, 64, 0, BF16) == 0


def test_kv_refusals(lib):
    st = (I64 * 4)(1024, 128, 1024, 128)

    def append(cache, rows=8, table=FAKE, tstride=4, cols=4, batch=2, max_len=4, dtype=BF16, k=FAKE, strides=st):
        return lib.mtq_kv_append(ctypes.byref(cache), k, FAKE, strides, rows, table, tstride, cols, FAKE, FAKE, FAKE, batch, max_len,
                                 dtype, None)

    def attend(cache, q=FAKE, rows=8, heads=32, table=FAKE, cols=4, batch=2, lq=1, lk=64, scale=0.1, dtype=BF16, ws=None, nb=0,
               strides=st):
        return lib.mtq_kv_attention(ctypes.byref(cache), q, FAKE, strides, rows, heads, table, cols, cols, FAKE, FAKE, FAKE, batch, lq,
                                    lk, 1, scale, dtype, ws, nb, None)

    for call in (append, attend):
        for bad in (dict(page_size=24), dict(page_size=8), dict(page_size=65536), dict(num_pages=0), dict(num_kv_heads=0),
                    dict(head_dim=96), dict(head_dim=512)):
            assert call(kv_cache(**bad)) == ARG, bad
        c = kv_cache()
        c.data[1] = 4104  # rows not 16-byte aligned
        assert call(c) == ARG
        c = kv_cache()
        c.data_strides[0][2] = 40
        assert call(c) == ARG
        c = kv_cache()
        c.scale[0] = None
        assert call(c) == ARG
        assert call(kv_cache(), table=None) == ARG
        assert call(kv_cache(), dtype=F64D) == DTYPE
        assert call(kv_cache(), rows=0) == OK and call(kv_cache(), batch=0) == OK
        assert call(kv_cache(), batch=-1) == ARG and call(kv_cache(), batch=70000) == ARG
        assert call(kv_cache(), cols=1 << 28) == ARG  # positions past 2^30
    assert append(kv_cache(), tstride=2) == ARG  # rows of the table overlap
    assert append(kv_cache(), k=None) == ARG
    assert attend(kv_cache(), heads=12) == ARG  # no multiple of the KV heads
    assert attend(kv_cache(), dtype=F32) == DTYPE
    assert attend(kv_cache(), scale=0.0) == ARG and attend(kv_cache(), scale=float("nan")) == ARG and attend(kv_cache(), scale=-1.0) == ARG
    assert attend(kv_cache(), strides=(I64 * 4)(1024, 130, 1024, 128)) == ARG
    need = lib.mtq_kv_attention_workspace_bytes(2, 32, 8, 128, 1, 4096)
    assert need > 0
    big = kv_cache(page_size=1024)
    assert attend(big, lk=4096) == ARG and attend(big, lk=4096, ws=FAKE, nb=need - 1) == ARG  # splits by the workspace


def test_python_refusals():
    x, w, s = torch.randn(4, 64), torch.zeros(16, 32, dtype=torch.uint8), torch.zeros(16, 2, dtype=torch.uint8)
    for call in (lambda f: mx_quantize(x, f), lambda f: mx_linear(x, w, s, format=f),
                 lambda f: rms_norm_quantize(x, torch.ones(64), format=f)):
        with pytest.raises(ValueError, match="format must be one of"):
            call("int4")
        with pytest.raises(RuntimeError, match="ROCm"):  # no CPU kernels
            call("mxfp8")
    with pytest.raises(NotImplementedError, match="head_dim"):
        NVFP4KVCache(2, 16, 1, 96, device="cpu")
    with pytest.raises(ValueError, match="page_size"):
        NVFP4KVCache(2, 24, 1, 128, device="cpu")
    c = NVFP4KVCache(2, 16, 1, 128, device="cpu")
    assert c.k_data.shape == (2, 1, 16, 64) and c.v_scale.dtype == torch.float8_e4m3fn and c.head_dim == 128
    with pytest.raises(ValueError, match="k_scale"):
        NVFP4KVCache.from_tensors(c.k_data, c.k_scale.view(torch.uint8), c.v_data, c.v_scale, c.k_amax, c.v_amax)
    with pytest.raises(ValueError, match="must both be"):
        NVFP4KVCache.from_tensors(c.k_data, c.k_scale, c.v_data[:1], c.v_scale, c.k_amax, c.v_amax)
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        c.attention(torch.randn(1, 1, 128), z, z, z, z.view(1, 1), 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        c.read(z, z, z, z.view(1, 1), 1, 1)


def test_mx_gemm_is_asked_for_and_kept():
    """Compressing as before computes as before; the choice travels with a saved model."""
    import io

    import modelopt_amd.torch.opt as mto
    import modelopt_amd.torch.quantization as mtq
    from modelopt_amd.torch.quantization import RealQuantLinear

    def model():
        torch.manual_seed(0)
        return torch.nn.Sequential(torch.nn.Linear(64, 32))

    for config, on in ((None, False), ({"quant_gemm": True}, False), ({"mx_gemm": True}, True), ({"mx_gemm": True, "quant_gemm": False}, False)):
        m = model()
        mtq.quantize(m, mtq.INT4_BLOCKWISE_WEIGHT_ONLY_CFG, lambda mm: mm(torch.ones(1, 64)))
        mtq.compress(m, config)
        assert isinstance(m[0], RealQuantLinear) and m[0]._use_mx_gemm is on
        buf = io.BytesIO()
        mto.save(m, buf)
        buf.seek(0)
        fresh = model()
        mto.restore(fresh, buf)
        assert fresh[0]._use_mx_gemm is on
        x = torch.randn(3, 64)
        with torch.no_grad():
            assert torch.equal(m(x), fresh(x))  # no packed product for this format: dequantised

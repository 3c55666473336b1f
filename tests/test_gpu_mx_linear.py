"""mx_quantize, rms_norm_quantize and mx_linear against the oracle's fake quants (bit for bit) and 64-bit sums.

Tolerance of the product, per element: operands are exact (E2M1 / E4M3 codes times powers of two), so y is off
by the fp32 sums, at most K rounding errors of 2^-23 (truncation counted) of the sum of magnitudes, and one
rounding to the output's type, eps / 2 of the value (half of the smallest subnormal below its normals). E4M3 by
E2M1 products are first added in groups of eight neighbours in fixed point, whose last bit is 2^-13 of
2^(the largest sum of exponents), cut toward zero. E2M1's 0.5 has the exponent of 1, every other code the one of
its own binade, so that bit is at most u = 2^-13 max|x| max(|w|, 1); the product that sets it has 6 significant
bits and is whole, the 7 others lose less than u each."""

import importlib

import pytest
import torch

from oracle import ref_ops as R

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ops():
    from modelopt_amd.torch.kernels import quantization as q

    return q


_VALUES = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def codes(packed):
    p = packed.cpu().long()
    return torch.stack((_VALUES[p % 16], _VALUES[p // 16]), -1).flatten(-2)


def values(data, scale, fmt):
    """What quantised rows stand for, in 64 bits on the CPU."""
    v = codes(data) if fmt == "mxfp4" else data.cpu().double()
    if fmt in ("mxfp4", "mxfp8"):
        return (v.unflatten(-1, (-1, 32)) * torch.exp2(scale.cpu().double() - 127).unsqueeze(-1)).flatten(-2)
    return v * scale.cpu().double()


def rows(m, k, dtype, seed=0, special=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    x[0, : min(32, k)] = 0
    x = x.to(dtype)
    if special and m > 3 and k >= 96:
        x[1, 3], x[1, 40], x[2, 70] = float("nan"), float("inf"), -float("inf")
        x[2, :32] = 2.0 ** -30 if dtype != torch.float16 else 2.0 ** -24
        x[3, 5] = -0.0
    return x


def packed_weight(n, k, seed, dev):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = torch.randint(115, 125, (n, k // 32), generator=g, dtype=torch.uint8)
    return w.to(dev), s.to(dev)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt,elem", [("mxfp4", "E2M1"), ("mxfp8", "E4M3")])
@pytest.mark.parametrize("m,k", [(1, 32), (5, 96), (33, 4096), (257, 160)])
def test_mx_quantize_is_the_fake_quant(gpu, dtype, fmt, elem, m, k):
    x = rows(m, k, DTYPES[dtype])
    data, scale = ops().mx_quantize(x.to(gpu), fmt)
    assert scale.dtype == torch.uint8 and scale.shape == (m, k // 32)
    want = R.fused_amax_convert(x, 32, elem)
    got = values(data, scale, fmt).to(x.dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(want.float()))


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_mx_quantize_extreme_blocks(gpu, dtype):
    """Blocks whose exponent is near either end of the type."""
    t = DTYPES[dtype]
    top, low = torch.finfo(t).max, torch.finfo(t).smallest_normal
    scales = [top, top / 3, low, low * 8, torch.finfo(t).tiny * 2 ** -5, 1.0]
    g = torch.Generator().manual_seed(1)
    x = torch.stack([(torch.rand(64, generator=g) * 2 - 1).double().mul(s).to(t) for s in scales])
    for fmt, elem in (("mxfp4", "E2M1"), ("mxfp8", "E4M3")):
        data, scale = ops().mx_quantize(x.to(gpu), fmt)
        want = R.fused_amax_convert(x, 32, elem)
        assert torch.equal(values(data, scale, fmt).to(t).float(), want.float()), (fmt, scale)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k", [8, 37, 1024])
def test_fp8_formats(gpu, dtype, k):
    x = rows(9, k, DTYPES[dtype], special=False)
    amax = torch.tensor([x.float().abs().amax() * 0.7])
    data, scale = ops().mx_quantize(x.to(gpu), "fp8", amax.to(gpu))
    assert data.dtype == torch.float8_e4m3fn and scale.shape == (1,)
    assert torch.equal((data.float() * scale).to(x.dtype).cpu(), R.fp8_eager(x, amax))
    data, scale = ops().mx_quantize(x.to(gpu), "fp8_token")
    want = x.float().abs().amax(-1, keepdim=True) / 448
    want[want == 0] = 1  # a row of zeros (k <= 32)
    assert torch.equal(scale.cpu(), want)
    got = values(data, scale, "fp8_token")
    # half a step of E4M3 (2^-4 of the value, 2^-10 of the factor below its normals), the factor's reciprocal rounded
    assert ((got - x.double()).abs() <= (2.0 ** -4 * x.double().abs() + 2.0 ** -10 * want.double()) * (1 + 2.0 ** -20)).all()


def test_mx_quantize_strides_and_empty(gpu):
    x = rows(12, 256, torch.bfloat16, special=False).to(gpu)
    want = ops().mx_quantize(x[:, 64:192].contiguous())
    for view in (x[:, 64:192], x.t().contiguous().t()[:, 64:192], x.view(3, 4, 256)[..., 64:192].reshape(3, 4, 128)):
        got = ops().mx_quantize(view)
        assert torch.equal(got[0].reshape(want[0].shape), want[0]) and torch.equal(got[1].reshape(want[1].shape), want[1])
    odd = torch.zeros(12 * 256 + 1, device=gpu, dtype=torch.bfloat16)[1:].view(12, 256)  # 2-byte aligned
    odd.copy_(x)
    assert torch.equal(ops().mx_quantize(odd)[0], ops().mx_quantize(x)[0])
    data, scale = ops().mx_quantize(x[:0])
    assert data.shape == (0, 128) and scale.shape == (0, 8)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8", "fp8", "fp8_token"])
@pytest.mark.parametrize("m,h,residual", [(1, 64, True), (3, 4096, True), (70, 160, False), (5, 2080, True), (2, 16416, True)])
def test_rms_norm_quantize(gpu, dtype, fmt, m, h, residual):
    t = DTYPES[dtype]
    g = torch.Generator().manual_seed(m + h)
    x = torch.randn(m, h, generator=g).to(t)
    r = (3 * torch.randn(m, h, generator=g)).to(t) if residual else None
    w = (1 + 0.3 * torch.randn(h, generator=g)).to(t if h != 4096 else torch.float32)
    x[0] = 0
    if residual:
        r[0] = 0
    hh = (x.double() + r.double()).to(t) if residual else x
    y = hh.double() * torch.rsqrt((hh.double() ** 2).mean(-1, keepdim=True) + 1e-5) * w.double()
    amax = y.abs().amax().float().reshape(1) * 0.8
    data, scale, h_out = ops().rms_norm_quantize(x.to(gpu), w.to(gpu), 1e-5, residual=r.to(gpu) if residual else None, format=fmt,
                                                 amax=amax.to(gpu) if fmt == "fp8" else None)
    if residual:
        assert torch.equal(h_out.cpu(), hh)
    else:
        assert h_out is None
    got = values(data, scale, fmt)
    if fmt in ("mxfp4", "mxfp8"):
        most, rel, step = (6.0, 0.25, 0.25) if fmt == "mxfp4" else (448.0, 2.0 ** -4, 2.0 ** -10)
        top = y.unflatten(-1, (-1, 32)).abs().amax(-1)
        e = scale.cpu().double() - 127
        ratio = top / (most * torch.exp2(e))  # in (1/2, 1] but for a rounding of y at the border; blocks of zeros: e = 0
        assert ((ratio <= 1 + 2.0 ** -22) & (ratio > 0.5 - 2.0 ** -23) | (top == 0) & (e == 0)).all()
        unit = torch.exp2(e).repeat_interleave(32, -1)
    else:
        rel, step = 2.0 ** -4, 2.0 ** -10
        unit = scale.cpu().double().expand_as(y) if fmt == "fp8_token" else torch.full_like(y, float(scale.item()))
    lim = y.clamp(-448 * unit, 448 * unit) if fmt == "fp8" else y
    # half a step (E2M1: a quarter of the value, 0.25 units near zero) and y's own fp32 rounding
    assert ((got - lim).abs() <= (rel * lim.abs() + step * unit) * (1 + 2.0 ** -20)).all()


def test_rms_norm_quantize_views_and_refusals(gpu):
    x = torch.randn(6, 3, 128, device=gpu).bfloat16()
    r = torch.randn(6, 3, 256, device=gpu).bfloat16()[..., ::2]  # strided columns: taken by a copy
    w = torch.ones(128, device=gpu).bfloat16()
    a = ops().rms_norm_quantize(x, w, residual=r)
    b = ops().rms_norm_quantize(x.reshape(18, 128), w, residual=r.contiguous().view(18, 128))
    for p, q in zip(a, b):
        assert torch.equal(p.reshape(q.shape).view(torch.uint8), q.view(torch.uint8))
    for bad, exc in ((dict(residual=r[:3]), ValueError), (dict(residual=r.float()), ValueError), (dict(format="fp8"), ValueError),
                     (dict(eps=-1.0), ValueError)):
        with pytest.raises(exc):
            ops().rms_norm_quantize(x, w, **{"eps": 1e-6, **bad}) if "eps" not in bad else ops().rms_norm_quantize(x, w, bad["eps"])
    with pytest.raises(ValueError):
        ops().rms_norm_quantize(x, w[:64])
    with pytest.raises(RuntimeError):
        ops().rms_norm_quantize(x, w.half())
    with pytest.raises(ValueError):
        ops().rms_norm_quantize(x[..., :40], w[:40])
    with pytest.raises(NotImplementedError):
        ops().rms_norm_quantize(x, w.clone().requires_grad_())


def product(xq, w, ws, bias):
    wv = (codes(w).unflatten(-1, (-1, 32)) * torch.exp2(ws.cpu().double().view(w.shape[0], -1) - 127).unsqueeze(-1)).flatten(-2)
    y = xq @ wv.t()
    one = torch.exp2(ws.cpu().double().view(w.shape[0], -1) - 127).repeat_interleave(4, -1)  # what |w| = 1 stands for
    most = torch.maximum(wv.abs().unflatten(-1, (-1, 8)).amax(-1), one)
    cut = 7 * 2.0 ** -13 * (xq.abs().unflatten(-1, (-1, 8)).amax(-1) @ most.t())
    return (y if bias is None else y + bias.cpu().double()), xq.abs() @ wv.abs().t(), cut


def check_product(y, xq, w, ws, bias, k, e4m3):
    want, mag, cut = product(xq, w, ws, bias)
    nan = torch.isnan(want)
    got = y.cpu().double()
    assert torch.equal(torch.isnan(got), nan)
    t = torch.finfo(y.dtype)
    tol = mag * k * 2.0 ** -23 + want.abs() * (t.eps / 2) * (1 + 2.0 ** -8) + t.smallest_normal * t.eps / 2
    if e4m3:
        tol = tol + cut * (1 + 2.0 ** -8)
    if bias is not None:
        tol = tol + bias.cpu().double().abs() * 2.0 ** -23
    # past the type's range (an infinity of x stands for 6 * 2^126 or more, alone in its row): infinity
    over = torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + tol >= t.max)
    assert (nan | over | ((got - want).abs() <= tol)).all(), ((got - want).abs() / tol)[~(nan | over)].max()


# rows that meet every form: streaming (1 .. 16), 64-row tiles, 128-row tiles, 256-row tiles; K and N that no tile divides
SHAPES = [(1, 16, 32), (1, 4096, 4096), (7, 33, 544), (8, 1000, 96), (16, 257, 4128), (16, 17000, 224), (17, 40, 32), (33, 100, 2080),
          (64, 300, 1696), (65, 129, 512), (200, 333, 160), (300, 8200, 416), (700, 6151, 288), (2100, 6500, 352),
          (2100, 6500, 96), (4300, 5001, 544)]


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8", "fp8", "fp8_token"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_mx_linear(gpu, fmt, m, n, k):
    dtype = torch.float16 if (m + n) % 3 == 0 else torch.bfloat16
    x = rows(m, k, dtype, seed=k, special=False)
    w, ws = packed_weight(n, k, m, gpu)
    bias = torch.randn(n, device=gpu).to(dtype if n % 2 else torch.float32) if m % 2 else None
    amax = (x.float().abs().amax() * 0.6).reshape(1).to(gpu) if fmt == "fp8" else None
    xg = x.to(gpu)
    y = ops().mx_linear(xg, w, ws, bias, format=fmt, amax=amax)
    assert y.shape == (m, n) and y.dtype == dtype
    data, scale = ops().mx_quantize(xg, fmt, amax)
    check_product(y, values(data, scale, fmt), w, ws, bias, k, fmt != "mxfp4")
    # handed over quantised, in the output type asked for
    for od in (torch.float32, dtype):
        z = ops().mx_linear(data, w, ws, bias if bias is None or bias.dtype in (od, torch.float32) else bias.to(od), format=fmt,
                            x_scale=scale, out_dtype=od)
        assert z.dtype == od
        check_product(z, values(data, scale, fmt), w, ws, bias, k, fmt != "mxfp4")


def test_mx_linear_special_values(gpu):
    """NaN and infinities in x: a row's own only (E2M1 has neither: NaN is +6, infinity the largest)."""
    for m in (4, 40, 300, 2100):
        for fmt in ("mxfp4", "mxfp8"):
            n = 200 if m < 1000 else 6500
            x = rows(m, 416, torch.bfloat16, special=True)
            w, ws = packed_weight(n, 416, 3, gpu)
            data, scale = ops().mx_quantize(x.to(gpu), fmt)
            v = values(data, scale, fmt)
            v, keep = v.clone(), ~torch.isnan(v).any(-1)
            y = ops().mx_linear(x.to(gpu), w, ws, format=fmt)
            check_product(y[keep.to(gpu)], v[keep], w, ws, None, 416, fmt == "mxfp8")
            assert torch.isnan(y[~keep.to(gpu)]).all()
            assert (~keep).sum() == (0 if fmt == "mxfp4" else 1)


def test_mx_linear_shapes_strides_and_refusals(gpu):
    x = torch.randn(3, 5, 192, device=gpu).bfloat16()
    w, ws = packed_weight(48, 128, 0, gpu)
    y = ops().mx_linear(x[..., 32:160], w, ws)
    assert y.shape == (3, 5, 48)
    z = ops().mx_linear(x[..., 32:160].contiguous().view(15, 128), w, ws)
    assert torch.equal(y.view(15, 48), z)
    assert torch.equal(z, ops().mx_linear(x[..., 32:160].reshape(15, 128), w.clone().t().contiguous().t(), ws.flatten()))
    odd = torch.zeros(48 * 64 + 1, device=gpu, dtype=torch.uint8)[1:].view(48, 64)
    odd.copy_(w)
    assert torch.equal(z, ops().mx_linear(x[..., 32:160].reshape(15, 128), odd, ws))
    assert ops().mx_linear(x[:0, :, :128], w, ws).shape == (0, 5, 48)
    d, s = ops().mx_quantize(x[..., :128].contiguous(), "mxfp8")
    for args, kw in (((x, w, ws), {}), ((x[..., :128], w.to(torch.int8), ws), {}), ((x[..., :128], w, ws[:40]), {}),
                     ((x[..., :128], w, ws, torch.zeros(47, device=gpu)), {}), ((d, w, ws), dict(x_scale=s, format="mxfp4")),
                     ((d, w, ws), dict(x_scale=s[:2], format="mxfp8")), ((x[..., :128], w, ws), dict(format="fp8")),
                     ((x[..., :128], w[:, :24], ws), {})):
        with pytest.raises(ValueError):
            ops().mx_linear(*args, **kw)
    with pytest.raises(RuntimeError):
        ops().mx_linear(x[..., :128].double(), w, ws)
    with pytest.raises(NotImplementedError):
        ops().mx_linear(x[..., :128].clone().requires_grad_(), w, ws)


def test_mx_linear_is_the_same_every_time(gpu):
    """Sums have a fixed order: any form gives the same bits again, on any stream, with other work between."""
    for m, n, k in ((3, 4096, 4096), (48, 4096, 4096), (500, 4096, 1696), (2100, 6500, 352)):
        x = torch.randn(m, k, device=gpu).bfloat16()
        w, ws = packed_weight(n, k, 1, gpu)
        a = ops().mx_linear(x, w, ws, format="mxfp8")
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            b = ops().mx_linear(x, w, ws, format="mxfp8")
        c = ops().mx_linear(x, w, ws, format="mxfp8")
        torch.cuda.current_stream().wait_stream(other)
        assert torch.equal(a, b) and torch.equal(a, c)


@pytest.mark.parametrize("m", [2, 40, 600, 2100])
def test_mx_linear_in_a_graph(gpu, m):
    n, k = (6500, 352) if m > 1000 else (4096, 1696)
    w, ws = packed_weight(n, k, 1, gpu)
    x = torch.randn(m, k, device=gpu).bfloat16()
    norm = torch.ones(k, device=gpu).bfloat16()

    def step():
        d, s, _ = ops().rms_norm_quantize(x, norm, format="mxfp8")
        return ops().mx_linear(d, w, ws, format="mxfp8", x_scale=s), ops().mx_linear(x, w, ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(m, k, device=gpu) * (i + 1))
        graph.replay()
        want = step()  # eager, between the replays
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), i


@pytest.mark.parametrize("preset,fmt", [("MXFP4_DEFAULT_CFG", "mxfp4"), ("W4A8_MXFP4_FP8_CFG", "fp8")])
def test_compressed_linear_computes_packed(gpu, preset, fmt, monkeypatch):
    """With mx_gemm a compressed MXFP4 model's linears run mx_linear; without it they dequantise, as they did."""
    import modelopt_amd.torch.quantization as mtq

    C = importlib.import_module("modelopt_amd.torch.quantization.compress")  # the package's own name is the function
    torch.manual_seed(0)
    calls = []
    real = C.mx_linear
    monkeypatch.setattr(C, "mx_linear", lambda *a, **k: (calls.append(k["format"]), real(*a, **k))[1])
    data = torch.randn(37, 256, device=gpu).bfloat16()
    for gemm in (True, False):
        torch.manual_seed(1)
        m = torch.nn.Sequential(torch.nn.Linear(256, 384), torch.nn.GELU(), torch.nn.Linear(384, 96, bias=False)).to(gpu).bfloat16()
        mtq.quantize(m, getattr(mtq, preset), lambda mm: mm(data))
        mtq.compress(m, {"mx_gemm": True} if gemm else None)
        calls.clear()
        with torch.no_grad():
            hidden = m[0](data)
            out = m[1:](hidden)
            m(data[:1].view(1, 1, 256))
            m(data[0])
        assert calls == ([fmt] * 6 if gemm else [])
        if gemm or fmt == "mxfp4":  # (the dequantised FP8 input is rounded once more)
            for layer, x, y in ((m[0], data, hidden), (m[2], m[1](hidden), out)):
                d, s = ops().mx_quantize(x, fmt, x.float().abs().amax().reshape(1) if fmt == "fp8" else None)
                check_product(y, values(d, s, fmt), layer.weight.data, layer.weight_quantizer._scale.view(layer.out_features, -1),
                              layer.bias, layer.in_features, fmt == "fp8")
        if gemm:  # a gradient, another dtype: dequantised
            calls.clear()
            m(data.clone().requires_grad_()).sum().backward()
            assert not calls

"""The packed operators at the ends of their ranges: rows of the smallest magnitudes, factors of the plain FP8
formats, lengths past their bounds, sizes past a launch's."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def ops():
    from modelopt_amd.torch.kernels import quantization as q

    return q


def token_codes(x):
    """The definition of FP8 per token: (codes as values, factors), by division in 32 bits."""
    a = torch.nan_to_num(x.float().abs(), nan=0.0, posinf=torch.finfo(torch.float32).max).amax(-1, keepdim=True)
    scale = a / 448
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return (x.float() / scale).clamp(-448, 448).to(torch.float8_e4m3fn).float(), scale


# ---- FP8 per token: codes of x / factor --------------------------------------------------------------------


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("k", [8, 37, 5000])
def test_fp8_token_rows_of_any_magnitude(gpu, dtype, k):
    """Rows whose largest value is anything the type holds: 1 / factor is past fp32 below 1.3e-36."""
    t = DTYPES[dtype]
    tops = [1.0, 3e-7, 2e-5, 6e4] + ([] if dtype == "fp16" else [1e-19, 2e-17, 1e-35, 1.3e-36, 1e-36, 1e-37, 1e-38, 3e-39, 1e-40, 1e30, 3e38])
    tops += [1e-44] if dtype == "fp32" else []
    g = torch.Generator().manual_seed(k)
    x = torch.stack([((2 * torch.rand(k, generator=g) - 1).double() * top).to(t) for top in tops])
    x[:, 1], x[:, 2] = 0.0, -0.0
    x[:, 0] = torch.tensor(tops).double().to(t)
    want, factor = token_codes(x)
    data, scale = ops().mx_quantize(x.to(gpu), "fp8_token")
    assert torch.equal(scale.cpu(), factor)
    assert torch.equal(data.cpu().float(), want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_fp8_token_codes_at_their_borders(gpu, dtype):
    """Every element is x / factor rounded once: 16-bit values of a wide row meet thousands of codes' borders."""
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(600, 4096, generator=g) * torch.exp(torch.randn(4096, generator=g))).to(DTYPES[dtype])
    want, factor = token_codes(x)
    data, scale = ops().mx_quantize(x.to(gpu), "fp8_token")
    assert torch.equal(scale.cpu(), factor) and torch.equal(data.cpu().float(), want)


def test_fp8_token_special_values(gpu):
    x = torch.randn(3, 64).bfloat16()
    x[0, 3], x[1, 4], x[2, 5], x[2, 6] = float("nan"), float("inf"), -float("inf"), float("nan")
    want, factor = token_codes(x)
    data, scale = ops().mx_quantize(x.to(gpu), "fp8_token")
    assert torch.equal(scale.cpu(), factor)
    assert torch.equal(torch.nan_to_num(data.cpu().float(), nan=1000.0), torch.nan_to_num(want, nan=1000.0))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("h", [64, 4096, 5001])
def test_rms_norm_fp8_token_of_small_weights(gpu, dtype, h):
    """y of 1e-36 and below: finite codes, zeros where y is zero, the factor of the row."""
    g = torch.Generator().manual_seed(h)
    x = torch.randn(4, h, generator=g).to(DTYPES[dtype])
    x[:, 5] = 0
    for small in (1e-35, 1e-36, 1e-37, 1e-38):
        w = (small * (1 + 0.3 * torch.randn(h, generator=g))).to(DTYPES[dtype])
        y = x.double() * torch.rsqrt((x.double() ** 2).mean(-1, keepdim=True) + 1e-5) * w.double()
        data, scale, _ = ops().rms_norm_quantize(x.to(gpu), w.to(gpu), 1e-5, format="fp8_token")
        f = scale.cpu().double()
        want = y.abs().amax(-1, keepdim=True) / 448
        # the factor: two fp32 roundings of y (three factors), one of the quotient; its own half step where it is subnormal
        assert ((f - want).abs() <= want * 2.0 ** -21 + 2.0 ** -149).all()
        got = data.cpu().double() * f
        # half a step of E4M3, y's three roundings (half a step of 2^-149 each where they are subnormal), saturation
        # where the factor was rounded down
        tol = (2.0 ** -4 * y.abs() + 2.0 ** -10 * f) * (1 + 2.0 ** -20) + 3 * 2.0 ** -149 + 448 * 2.0 ** -149
        assert ((got - y).abs() <= tol).all()
        assert (got[:, 5] == 0).all()


def test_mx_linear_fp8_token_rows_of_small_magnitude(gpu):
    from test_gpu_mx_linear import check_product, packed_weight, values

    for m, n, k in ((3, 48, 512), (40, 96, 256), (300, 260, 288)):
        x = torch.randn(m, k).double()
        x[1] *= 1e-37
        x[2] *= 3e-38
        x[:, 7] = 0
        x = x.bfloat16().to(gpu)
        w, ws = packed_weight(n, k, m, gpu)
        data, scale = ops().mx_quantize(x, "fp8_token")
        y = ops().mx_linear(x, w, ws, format="fp8_token", out_dtype=torch.float32)
        assert torch.isfinite(y).all()
        check_product(y, values(data, scale, "fp8_token"), w, ws, None, k, True)

"""The operators of a packed 4-bit model's decoder layer, as cases to be measured: the RMS norm that quantises its output,
the product with microscaled 4-bit weights, and the KV cache held in 4 bits with its attention.

With ``own`` false ``run`` computes them with elementary torch operations in 32 bits; with ``own`` true it makes the calls
that a user of ``modelopt_amd`` makes."""

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@functools.lru_cache(maxsize=1)
def _product():
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tensorrt-model-optimizer_amd"))
    from modelopt_amd.torch.kernels.common.attention import NVFP4KVCache
    from modelopt_amd.torch.kernels.quantization import mx_linear, rms_norm_quantize

    return mx_linear, rms_norm_quantize, NVFP4KVCache


# ---- cases ------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # the output projection of a Llama-3-8B layer while one user's answer is generated: latency
        _linear("linear w4a4 one token", 1, 4096, 4096, "mxfp4", "bf16"),
        # the widest projection of Llama-3-70B for a batch of decoding users, activations in 8 bits
        _linear("linear w4a8 decode batch", 48, 28672, 8192, "mxfp8", "bf16"),
        # the up projection of Llama-3-8B over a calibration batch or a long prompt
        _linear("linear w4a4 prompt", 8192, 14336, 4096, "mxfp4", "bf16"),
        # W4A8_MXFP4_FP8: static FP8 activations, a bias, and sizes that no tile divides
        _linear("linear w4a8 ragged", 1531, 6151, 1696, "fp8", "fp16", bias=True),
        # the norm before a projection in a decode step of 16 users
        _norm("norm decode batch", 16, 4096, "mxfp8", "bf16", True),
        # the same over the 32 x 512 tokens of a calibration batch
        _norm("norm prompt", 16384, 4096, "mxfp8", "bf16", True),
        # one scale per token, a first norm (no residual yet), a width that no block divides
        _norm("norm per token ragged", 2501, 5000, "fp8_token", "fp16", False),
        # one new token for each of 32 users into the cache, and its rows read back
        _cache("cache step", "append", 32, 1, 1, 2000, 8, 8, 128, 16, "bf16"),
        # prompts of unequal lengths written behind earlier context, and read back for the prompt's own attention
        _cache("cache prompt", "append", 7, 900, 6000, 8000, 8, 8, 128, 64, "bf16"),
        # one user, a short answer: latency
        _cache("attention one user", "attention", 1, 1, 1, 1000, 32, 8, 128, 16, "bf16"),
        # 64 users with contexts up to 16384 tokens, Llama-3-8B's heads: the cache's bytes count
        _cache("attention decode batch", "attention", 64, 1, 1, 16384, 32, 8, 128, 64, "bf16"),
        # chunks of prompts over the context before them
        _cache("attention chunk", "attention", 4, 500, 1024, 8192, 32, 8, 128, 64, "bf16"),
    ]


def _linear(name, m, n, k, fmt, dtype, bias=False):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "fmt": fmt, "dtype": dtype, "bias": bias}


def _norm(name, rows, width, fmt, dtype, residual):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "fmt": fmt, "dtype": dtype, "residual": residual}


def _cache(name, op, batch, q_min, q_max, kv_max, heads, kv_heads, head_dim, page, dtype):
    """Sequences of q_min .. q_max new tokens at the end of contexts of up to kv_max tokens (the new ones among them)."""
    return {"name": name, "op": op, "batch": batch, "q_min": q_min, "q_max": q_max, "kv_max": kv_max, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page": page, "dtype": dtype}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    kind = rng.choice(["linear", "linear", "norm", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "linear":
        m, n, k = _log(rng, 1, 8192), _log(rng, 256, 28672), 32 * _log(rng, 16, 448)
        while m * n * k > 8192 * 14336 * 4096:
            m = max(1, m // 2)
        c = _linear("", m, n, k, rng.choice(["mxfp4", "mxfp8", "fp8"]), dtype, rng.random() < 0.3)
    elif kind == "norm":
        fmt = rng.choice(["mxfp8", "fp8_token"])
        width = 32 * _log(rng, 16, 512) if fmt == "mxfp8" else _log(rng, 512, 16384)
        c = _norm("", max(1, min(_log(rng, 1, 32768), 16384 * 4096 // width)), width, fmt, dtype, rng.random() < 0.7)
    elif kind == "append":
        batch, q = _log(rng, 1, 64), _log(rng, 1, 4096)
        q = max(1, min(q, 40000 // batch))
        c = _cache("", "append", batch, max(1, q // 3), q, q + _log(rng, 1, 4096), 8, rng.choice([1, 2, 8]), rng.choice([64, 128]),
                   rng.choice([16, 32, 64]), dtype)
    else:
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 4, 5, 8])
        head_dim = rng.choice([64, 128])
        if rng.random() < 0.6:  # decode, sometimes a few tokens at once
            q = rng.choice([1, 1, 1, 2, 5])
            batch, kv = _log(rng, 1, 64), _log(rng, 16, 16384)
        else:
            q = _log(rng, 16, 1024)
            batch, kv = rng.choice([1, 2, 3]), q + _log(rng, 1, 6000)
            heads = kv_heads * rng.choice([1, 4])
        c = _cache("", "attention", batch, max(1, q // 2), q, max(kv, q), heads, kv_heads, head_dim, rng.choice([16, 32, 64]), dtype)
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, context with them) of every sequence: plain numbers that go by the case's sizes."""
    r = random.Random(case["batch"] * 7919 + case["q_max"] * 104729 + case["kv_max"])
    q = [r.randint(case["q_min"], case["q_max"]) for _ in range(case["batch"])]
    kv = [max(n, r.randint(max(1, case["kv_max"] // 4), case["kv_max"])) for n in q]
    q[0], kv[0] = case["q_max"], case["kv_max"]
    return q, kv


def work(case):
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": 2 * m * k + n * k * 17 / 32 + 2 * m * n + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        scales = n / 32 if case["fmt"] == "mxfp8" else 4 * case["rows"]
        return {"bytes": (2 + 2 * case["residual"] * 2 + 1) * n + scales + 2 * case["width"], "flops": 8 * n}
    q, kv = (sum(n) for n in _lengths(case))
    row = case["kv_heads"] * case["head_dim"]
    if case["op"] == "append":
        return {"bytes": 2 * q * row * (2 + 9 / 16 + 2), "flops": 2 * q * row * 6}
    pairs = sum(n * (c - n) + n * (n + 1) / 2 for n, c in zip(*_lengths(case)))
    qo = 2 * 2 * q * case["heads"] * case["head_dim"]
    return {"bytes": 2 * kv * row * 9 / 16 + qo, "flops": 4 * pairs * case["heads"] * case["head_dim"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    g = _gen(seed)
    dtype = _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        # activations as a norm leaves them: some channels carry far larger values than others
        channel = torch.exp(0.6 * _randn(g, k))
        s["x"] = (_randn(g, m, k) * channel).to(dtype)
        # the packed weight of a compressed model: codes of two columns in a byte (the even one low), an exponent per 32
        s["w"], s["w_scale"] = _pack_mxfp4(_randn(g, n, k) * (k ** -0.5))
        s["bias"] = _randn(g, n).to(dtype) if case["bias"] else None
        s["amax"] = torch.full((1,), 20.0, device=DEV) if case["fmt"] == "fp8" else None  # calibrated: a few values saturate
    elif case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        channel = torch.exp(0.6 * _randn(g, width))
        s["x"] = _randn(g, rows, width).to(dtype)
        s["r"] = (2 * _randn(g, rows, width) * channel).to(dtype) if case["residual"] else None
        s["w"] = (1 + 0.2 * _randn(g, width)).to(dtype)
    else:
        s.update(_prepare_cache(case, g, dtype))
    return s


def _pack_mxfp4(w):
    n, k = w.shape
    code, e = _mx_block(w.view(n, k // 32, 32), 6.0)
    q = _e2m1_code(code).view(n, k)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8)


def _prepare_cache(case, g, dtype):
    q_len, kv_len = _lengths(case)
    page, hkv, d = case["page"], case["kv_heads"], case["head_dim"]
    used = [-(-n // page) for n in kv_len]
    spare = 3  # a cache has free pages
    pages = sum(used) + spare
    order = torch.randperm(pages, generator=g, device=DEV).int()  # pages are handed out in no order
    table = torch.zeros(len(used), max(used), dtype=torch.int32)
    at = 0
    order = order.cpu()
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    start = [sum(q_len[:b]) for b in range(len(q_len))]

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    s = {"table": table.to(DEV), "start": ints(start), "q_len": ints(q_len), "kv_len": ints(kv_len), "q_max": case["q_max"],
         "kv_max": case["kv_max"], "tokens": sum(q_len),
         # calibrated over other prompts: no round numbers
         "k_amax": 9 + 4 * torch.rand(1, generator=g, device=DEV), "v_amax": 4 + torch.rand(1, generator=g, device=DEV)}
    if case["op"] == "append":
        shape = (sum(q_len), hkv, d)
        s["k"] = (_randn(g, *shape) * torch.exp(0.4 * _randn(g, d))).to(dtype)
        s["v"] = _randn(g, *shape).to(dtype)
        for n in ("k", "v"):
            s[n + "_data"] = torch.zeros(pages, hkv, page, d // 2, dtype=torch.uint8, device=DEV)
            s[n + "_scale"] = torch.zeros(pages, hkv, page, d // 16, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        return s
    # a filled cache: keys with channels of unequal size, rotated or not, look normal to the attention
    for n in ("k", "v"):
        rows = _randn(g, pages * hkv * page, d)
        if n == "k":
            rows = rows * torch.exp(0.4 * _randn(g, d))
        code, scale = _nvfp4_block(rows, s[n + "_amax"])
        s[n + "_data"] = _pair(code).view(pages, hkv, page, d // 2)
        s[n + "_scale"] = scale.view(pages, hkv, page, d // 16)
        del rows, code, scale
    s["q"] = _randn(g, sum(q_len), case["heads"], d).to(dtype)
    return s


# ---- plain forms ------------------------------------------------------------------------------------------------------

_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _e2m1_round(v):
    """The nearest value of 0, .5, 1, 1.5, 2, 3, 4, 6 with v's sign; halves to the even code; 6 beyond."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), v)


def _e2m1_code(v):
    """The 4-bit code of an E2M1 value."""
    a = v.abs()
    mag = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4))
    return mag.to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)


def _e2m1_value(packed):
    """[..., n] bytes -> [..., 2n] values in 32 bits, the low half of a byte first."""
    lut = torch.tensor(_E2M1, device=packed.device)
    return torch.stack((lut[(packed & 15).int()], lut[(packed >> 4).int()]), -1).flatten(-2)


def _exponent(ratio):
    """ceil(log2(ratio)) for ratio > 0, 0 for 0."""
    m, e = torch.frexp(ratio)
    e = torch.where(m > 0.5, e, e - 1).clamp(-127, 127)
    return torch.where(ratio > 0, e, torch.zeros_like(e))


def _mx_block(x, most):
    """Blocks in the last axis, 32 bits: (x / 2^e rounded to the format whose largest value is ``most``, e [..., 1])."""
    e = _exponent(x.abs().amax(-1) / torch.tensor(most, device=x.device))
    v = torch.ldexp(x, -e.unsqueeze(-1))
    return (_e2m1_round(v) if most == 6.0 else v.clamp(-448, 448).to(torch.float8_e4m3fn).float()), e


def _nvfp4_block(x, amax):
    """Rows [n, d] in 32 bits: (E2M1 values [n, d], e4m3 scale per 16 [n, d / 16])."""
    gs = amax / torch.tensor(2688.0, device=x.device)
    b = x.view(x.shape[0], -1, 16)
    s8 = (b.abs().amax(-1) / (6.0 * gs)).clamp(max=448.0).to(torch.float8_e4m3fn)
    q = s8.float() * gs
    dead = q < 1e-5
    v = _e2m1_round(b / torch.where(dead, torch.ones_like(q), q).unsqueeze(-1))
    return v.view(x.shape), torch.where(dead, torch.zeros_like(q), s8.float()).to(torch.float8_e4m3fn)


def _pair(values):
    c = _e2m1_code(values)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def _plain_linear(s):
    case, x = s["case"], s["x"].float()
    m, n, k = case["m"], case["n"], case["k"]
    if case["fmt"] == "fp8":
        scale = 448.0 / s["amax"]
        xq = (x * scale).clamp(-448, 448).to(torch.float8_e4m3fn).float() / scale
    else:
        v, e = _mx_block(x.view(m, k // 32, 32), 6.0 if case["fmt"] == "mxfp4" else 448.0)
        xq = torch.ldexp(v, e.unsqueeze(-1)).view(m, k)
    w = _e2m1_value(s["w"]).view(n, k // 32, 32)
    w = torch.ldexp(w, s["w_scale"].int().unsqueeze(-1) - 127).view(n, k)
    y = xq @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_norm(s):
    case, x = s["case"], s["x"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5) * s["w"].float()
    if case["fmt"] == "mxfp8":
        v, e = _mx_block(y.view(y.shape[0], -1, 32), 448.0)
        return h, v.view(y.shape).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)
    amax = y.abs().amax(-1, keepdim=True)
    scale = torch.where(amax > 0, amax / torch.tensor(448.0, device=x.device), torch.ones_like(amax))
    return h, (y / scale).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _token_places(s):
    """For every new token: its sequence, its page and its place in the page."""
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["start"], t, right=True) - 1
    pos = t - s["start"][b] + s["kv_len"][b] - s["q_len"][b]
    page = s["case"]["page"]
    return b, s["table"][b, pos // page].long(), (pos % page).long()


def _plain_append(s):
    _, page, place = _token_places(s)
    out = []
    for n in ("k", "v"):
        x = s[n]
        t, h, d = x.shape
        code, scale = _nvfp4_block(x.float().view(t * h, d), s[n + "_amax"])
        s[n + "_data"][page, :, place] = _pair(code).view(t, h, d // 2)
        s[n + "_scale"].view(torch.uint8)[page, :, place] = scale.view(torch.uint8).view(t, h, d // 16)
        v = _e2m1_value(s[n + "_data"][page, :, place]).view(t, h, d // 16, 16)
        gs = s[n + "_amax"] / torch.tensor(2688.0, device=x.device)
        q = s[n + "_scale"].view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn).float() * gs
        out.append((v * q.unsqueeze(-1)).view(t, h, d).to(x.dtype))
    return out


def _plain_attention(s):
    case, q = s["case"], s["q"].float()
    hkv, d, page = case["kv_heads"], case["head_dim"], case["page"]
    group = case["heads"] // hkv
    batch, slots = s["table"].shape
    kv = {}
    for n in ("k", "v"):  # [B, slots, Hkv, page, D] -> [B, Hkv, keys, D]
        table = s["table"].long()
        x = _e2m1_value(s[n + "_data"][table]).view(batch, slots, hkv, page, d // 16, 16)
        x = x * (s[n + "_scale"].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * (s[n + "_amax"] / 2688.0)).unsqueeze(-1)
        kv[n] = x.view(batch, slots, hkv, page, d).permute(0, 2, 1, 3, 4).reshape(batch, hkv, slots * page, d)
    rows = torch.arange(s["q_max"], device=DEV, dtype=torch.int32)
    at = (s["start"][:, None] + rows).clamp(max=s["tokens"] - 1).long()  # padded rows: any token, dropped below
    qp = q[at].view(batch, s["q_max"], hkv, group, d).permute(0, 2, 3, 1, 4).reshape(batch, hkv, group * s["q_max"], d)
    score = torch.matmul(qp, kv["k"].transpose(2, 3)).view(batch, hkv, group, s["q_max"], -1) * d ** -0.5
    key = torch.arange(slots * page, device=DEV, dtype=torch.int32)
    last = (s["kv_len"] - s["q_len"])[:, None] + rows  # a query sees the keys up to its own place
    score = score.masked_fill((key > last[..., None])[:, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = torch.matmul((p / p.sum(-1, keepdim=True)).view(batch, hkv, group * s["q_max"], -1), kv["v"])
    o = o.view(batch, hkv, group, s["q_max"], d).permute(0, 3, 1, 2, 4).reshape(batch, s["q_max"], hkv * group, d)
    t = torch.arange(s["tokens"], device=DEV, dtype=torch.int32)
    b = torch.searchsorted(s["start"], t, right=True) - 1
    return o[b, (t - s["start"][b]).long()].to(s["q"].dtype)


# ---- one pass ---------------------------------------------------------------------------------------------------------


def _own(s):
    mx_linear, rms_norm_quantize, NVFP4KVCache = _product()
    case = s["case"]
    if case["op"] == "linear":
        return mx_linear(s["x"], s["w"], s["w_scale"], s["bias"], format=case["fmt"], amax=s["amax"])
    if case["op"] == "norm":
        q, scale, h = rms_norm_quantize(s["x"], s["w"], 1e-5, residual=s["r"], format=case["fmt"])
        return (s["x"] if h is None else h), q, (scale.view(torch.float8_e8m0fnu) if case["fmt"] == "mxfp8" else scale)
    if "cache" not in s:  # the handle that a program keeps for its cache's memory
        s["cache"] = NVFP4KVCache.from_tensors(s["k_data"], s["k_scale"], s["v_data"], s["v_scale"], s["k_amax"], s["v_amax"])
    cache = s["cache"]
    if case["op"] == "append":
        cache.append(s["k"], s["v"], s["start"], s["q_len"], s["kv_len"], s["table"], s["q_max"])
        return list(cache.read(s["start"], s["q_len"], s["kv_len"], s["table"], s["q_max"], s["tokens"], dtype=s["k"].dtype))
    return cache.attention(s["q"], s["start"], s["q_len"], s["kv_len"], s["table"], s["q_max"], s["kv_max"])


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "linear":
        return _plain_linear(state)
    if op == "norm":
        return _plain_norm(state)
    return _plain_append(state) if op == "append" else _plain_attention(state)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------


def _x_pow2_ceil(r):
    """2^ceil(log2 r), 1 where r is 0."""
    return torch.where(r > 0, torch.exp2(torch.ceil(torch.log2(torch.where(r > 0, r, 1.0)))), 1.0)


def _x_grid(v, mantissa, emin, most):
    """v rounded to the nearest number of a small floating format, halves to even, saturating."""
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** (emin - 2)))).clamp(min=emin)
    quantum = torch.exp2(e - mantissa)
    return (torch.round(v / quantum) * quantum).clamp(-most, most)


def _x_codes(packed):
    c = torch.stack((packed % 16, packed // 16), -1).flatten(-2).long()
    e, f = (c % 8) // 2, (c % 2).double()
    mag = torch.where(e == 0, f / 2, (1 + f / 2) * torch.exp2((e - 1).double()))
    return torch.where(c >= 8, -mag, mag)


def _x_cache_rows(s, n, page, place):
    """Rows of the cache at (page, place) of every head: [tokens, heads, d]."""
    v = _x_codes(s[n + "_data"][page, :, place])
    sc = s[n + "_scale"].view(torch.uint8)[page, :, place].view(torch.float8_e4m3fn).double() * (s[n + "_amax"].double() / 2688)
    return (v.unflatten(-1, (-1, 16)) * sc[..., None]).flatten(-2)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x = s["x"].double()
        if case["fmt"] == "fp8":
            f = 448 / s["amax"].double()
            x = _x_grid((x * f).clamp(-448, 448), 3, -6, 448) / f
        else:
            b = x.unflatten(-1, (-1, 32))
            u = _x_pow2_ceil(b.abs().amax(-1, keepdim=True) / (6 if case["fmt"] == "mxfp4" else 448))
            x = ((_x_grid(b / u, 1, 0, 6.0) if case["fmt"] == "mxfp4" else _x_grid(b / u, 3, -6, 448.0)) * u).flatten(-2)
        w = (_x_codes(s["w"]).unflatten(-1, (-1, 32)) * torch.exp2(s["w_scale"].double() - 127)[..., None]).flatten(-2)
        y = x @ w.t().contiguous()
        return y if s["bias"] is None else y + s["bias"].double()
    if case["op"] == "norm":
        h = s["x"].double() if s["r"] is None else (s["x"].double() + s["r"].double()).to(s["x"].dtype).double()
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-5) * s["w"].double()
        if case["fmt"] == "mxfp8":
            b = y.unflatten(-1, (-1, 32))
            u = _x_pow2_ceil(b.abs().amax(-1, keepdim=True) / 448)
            return h, _x_grid(b / u, 3, -6, 448.0).flatten(-2), u[..., 0]
        sc = y.abs().amax(-1, keepdim=True) / 448
        return h, _x_grid(y / sc, 3, -6, 448.0), sc
    q_len, kv_len = _lengths(case)
    if case["op"] == "append":
        out = []
        for n in ("k", "v"):
            b = s[n].double().unflatten(-1, (-1, 16))
            gs = s[n + "_amax"].double() / 2688
            sc = _x_grid((b.abs().amax(-1, keepdim=True) / (6 * gs)).clamp(max=448), 3, -6, 448.0) * gs
            out.append(torch.where(sc >= 1e-5, _x_grid(b / sc, 1, 0, 6.0) * sc, 0.0).flatten(-2))
        return out
    out = torch.empty(sum(q_len), case["heads"], case["head_dim"], dtype=torch.float64, device=DEV)
    at = 0
    for i, (n, c) in enumerate(zip(q_len, kv_len)):
        pos = torch.arange(c, device=DEV)
        page, place = s["table"][i].long()[pos // case["page"]], pos % case["page"]
        k, v = (_x_cache_rows(s, name, page, place).transpose(0, 1) for name in ("k", "v"))  # [Hkv, keys, D]
        q = s["q"][at:at + n].double().unflatten(1, (case["kv_heads"], -1)).permute(1, 2, 0, 3)  # [Hkv, G, n, D]
        score = torch.matmul(q.flatten(1, 2), k.transpose(1, 2).contiguous()).view(*q.shape[:3], c) / math.sqrt(case["head_dim"])
        hidden = pos[None, :] > torch.arange(c - n, c, device=DEV)[:, None]
        p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        o = torch.matmul(p.flatten(1, 2), v.contiguous()).view(q.shape)
        out[at:at + n] = o.permute(2, 0, 1, 3).flatten(1, 2)
        at += n
    return out

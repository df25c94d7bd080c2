"""Workloads of the norm-and-quantise operator and of the 4-bit floating-point operators.

Four operators: ``norm`` (RMS norm of the sum of an activation and the residual stream, with an 8-bit output),
``quantise`` (microscaled 4-bit floating point), ``product`` (matrix product of two such operands with the
linear layer's epilogue) and ``linear`` (a float activation through a layer with 4-bit weights).

With ``own`` false, ``run`` evaluates the operators in their plain form, elementary torch operations in 32 bits;
with ``own`` true it makes the calls of ``sam_quantization_b200.ops``.  ``exact`` restates the definitions in
64 bits.

The storage of a 4-bit operand [rows, K], in blocks of 32 (``mxfp4``) or 16 (``nvfp4``) columns:
  codes  uint8 [rows, pitch]: two e2m1 codes a byte, the even column in the low nibble; pitch = ceil(K/2) up to 16
  scales uint8 [ceil(rows/128), G, 32, 4, 4]: the scale byte of (row, block) at
         [row // 128, block // 4, row % 32, row % 128 // 32, block % 4], G = 4-block groups of ceil(K/256)*256 columns.
"""
import math

import torch

own = False

EPS = 1e-6
BLOCK = {"mxfp4": 32, "nvfp4": 16}
DTYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
LARGEST = 32768 * 5120                 # elements of the largest activation
LARGEST_PRODUCT = 32768 * 1280 * 5120  # multiply-adds of the largest product


# ---- the cases ------------------------------------------------------------------------------------

def _norm(M, K, dtype, residual):
    return {"op": "norm", "M": M, "K": K, "dtype": dtype, "residual": residual}


def _quantise(M, K, dtype, fmt, glob):
    return {"op": "quantise", "M": M, "K": K, "dtype": dtype, "fmt": fmt, "global_scale": glob}


def _product(M, N, K, dtype, fmt, bias, gelu, residual):
    return {"op": "product", "M": M, "N": N, "K": K, "dtype": dtype, "fmt": fmt, "bias": bias, "gelu": gelu, "residual": residual}


def _linear(M, N, K, dtype, fmt, bias, gelu, residual):
    return {"op": "linear", "M": M, "N": N, "K": K, "dtype": dtype, "fmt": fmt, "bias": bias, "gelu": gelu, "residual": residual}


def listed():
    return [
        # one new token of a width-1280 block: latency of the call
        dict(_norm(1, 1280, "bf16", True), name="norm: one token"),
        # eight images of 64 x 64 tokens in front of qkv
        dict(_norm(32768, 1280, "fp16", True), name="norm: 8 images"),
        # a ragged batch of an odd width, no residual (the first norm of a network)
        dict(_norm(4901, 1023, "bf16", False), name="norm: odd width"),
        # the windows of one image (25 windows of 14 x 14 tokens) in front of qkv
        dict(_quantise(4900, 1280, "fp16", "nvfp4", False), name="quantise: windows of an image"),
        # the hidden activations of the MLP of eight images
        dict(_quantise(32768, 5120, "bf16", "mxfp4", False), name="quantise: MLP hidden"),
        # a float weight of odd sizes with a global scale, as a layer is converted
        dict(_quantise(3001, 1283, "fp32", "nvfp4", True), name="quantise: odd weight"),
        # a few tokens against qkv-sized weights: latency and the weight's bytes
        dict(_product(8, 3840, 1280, "bf16", "nvfp4", True, False, False), name="product: 8 tokens"),
        # eight images through the first MLP linear with its GELU
        dict(_product(32768, 5120, 1280, "fp16", "nvfp4", True, True, False), name="product: MLP up"),
        # eight images through the second MLP linear, onto the residual stream
        dict(_product(32768, 1280, 5120, "bf16", "mxfp4", True, False, True), name="product: MLP down"),
        # one new token through an MLP linear: the serving form
        dict(_linear(1, 5120, 1280, "bf16", "nvfp4", True, True, False), name="linear: one token"),
        # one 14 x 14 window through qkv
        dict(_linear(196, 2304, 768, "fp16", "mxfp4", True, False, False), name="linear: one window"),
        # ragged everything: a padded batch through a layer of odd sizes
        dict(_linear(2777, 1001, 1283, "fp16", "nvfp4", True, False, True), name="linear: odd sizes"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "quantise", "product", "linear"))
    M = _log(rng, 1, 32768)
    fmt = rng.choice(("mxfp4", "nvfp4"))
    half = rng.choice(("fp16", "bf16"))
    if op == "norm":
        return _norm(M, min(_log(rng, 16, 8192), LARGEST // M), half, rng.random() < 0.7)
    if op == "quantise":
        return _quantise(M, min(_log(rng, 16, 8192), LARGEST // M), rng.choice(("fp16", "bf16", "fp32")), fmt, fmt == "nvfp4" and rng.random() < 0.5)
    K = _log(rng, 32, 5120)
    if rng.random() < 0.5:
        K = max(64, K // 64 * 64)
    N = max(1, min(_log(rng, 8, 5120), LARGEST_PRODUCT // (M * K)))
    make = _product if op == "product" else _linear
    return make(M, N, K, half, fmt, rng.random() < 0.7, rng.random() < 0.3, rng.random() < 0.4)


# ---- the 4-bit format, plain ------------------------------------------------------------------------

def _pad_columns(x, multiple):
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % multiple))


def _blocks(x, fmt):
    """[rows, K] -> fp32 [rows, blocks, block], zeros behind K."""
    b = BLOCK[fmt]
    return _pad_columns(x.float(), b).unflatten(-1, (-1, b))


def _power_of_two(byte):
    """2^(byte - 127) of int32 bytes 0..254, exactly (2^-127 is subnormal in 32 bits)."""
    return torch.where(byte > 0, byte << 23, 1 << 22).view(torch.float32)


def _quantise_plain(x, fmt, glob):
    """(values of the e2m1 codes [rows, blocks, block], block scales without the global one [rows, blocks, 1],
    block scales with it), fp32."""
    xb = _blocks(x, fmt)
    amax = xb.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        byte = ((amax.view(torch.int32) >> 23) - 2).clamp(min=0)
        own_scale = scale = _power_of_two(byte)
        v = xb * ((254 - byte) << 23).view(torch.float32)
    else:
        # a power of two for glob keeps every border times a scale exact, so that 32 bits decide as 64 do
        own_scale = (amax / torch.full((1,), 6.0 * glob, device=x.device)).clamp(max=448.0).to(torch.float8_e4m3fn).float().clamp(min=2.0 ** -9)
        scale = own_scale * glob
        v = xb / scale
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign((torch.round(a / step) * step).clamp(max=6.0), xb), own_scale, scale


def _store(values, own_scale, fmt, K):
    """The stored operand (codes, scales) of _quantise_plain's values and scales."""
    rows = values.shape[0]
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=values.device)
    code = torch.searchsorted(table, values.abs()).to(torch.uint8) + 8 * torch.signbit(values).to(torch.uint8)
    code = code.flatten(1)[:, :K]
    code = _pad_columns(code, 32)
    codes = code[:, 0::2] + 16 * code[:, 1::2]
    if fmt == "mxfp4":
        byte = (own_scale.view(torch.int32) >> 23).to(torch.uint8)
    else:
        byte = own_scale.to(torch.float8_e4m3fn).view(torch.uint8)
    byte = byte[..., 0]
    groups = 256 // BLOCK[fmt] // 4 * (-(-K // 256))
    byte = torch.nn.functional.pad(byte, (0, 4 * groups - byte.shape[1], 0, -rows % 128))
    return codes.contiguous(), byte.view(-1, 4, 32, groups, 4).permute(0, 3, 2, 1, 4).contiguous()


def _load(codes, scales, fmt, rows, K):
    """fp32 [rows, K] of a stored operand, without its global scale."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    table = torch.cat((table, -table))
    v = table[torch.stack((codes & 15, codes >> 4), -1).flatten(1).long()[:, :K]]
    byte = scales.permute(0, 3, 2, 1, 4).reshape(-1, 4 * scales.shape[1])[:rows, : -(-K // BLOCK[fmt])]
    s = _power_of_two(byte.int()) if fmt == "mxfp4" else byte.contiguous().view(torch.float8_e4m3fn).float()
    return (_blocks(v, fmt) * s[..., None]).flatten(1)[:, :K]


# ---- the operators, plain ---------------------------------------------------------------------------

def _norm_plain(s):
    x, r = s["x"], s["residual"]
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    scale = y.abs().amax(-1, keepdim=True).clamp(min=1e-5) / torch.full((1,), 127.0, device=x.device)
    out = {"values": (torch.round(y / scale) * scale).to(x.dtype), "scale": scale[:, 0]}
    return out if r is None else dict(out, residual=h)


def _epilogue_plain(acc, s):
    y = acc
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["gelu"]:
        y = 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["dtype"])


def _run_plain(s):
    if s["op"] == "norm":
        return _norm_plain(s)
    if s["op"] == "quantise":
        v, _, scale = _quantise_plain(s["x"], s["fmt"], s["x_global"])
        return {"values": (v * scale).flatten(1)[:, : s["K"]].to(s["x"].dtype)}
    if s["op"] == "product":
        a = _load(s["x_codes"], s["x_scales"], s["fmt"], s["M"], s["K"])
    else:
        v, _, scale = _quantise_plain(s["x"], s["fmt"], 1.0)
        a = (v * scale).flatten(1)[:, : s["K"]]
    acc = a @ _load(s["w_codes"], s["w_scales"], s["fmt"], s["N"], s["K"]).t()
    return {"y": _epilogue_plain(acc * s["w_global"], s)}


# ---- the framework's calls --------------------------------------------------------------------------

def _run_own(s):
    from sam_quantization_b200 import ops
    if s["op"] == "norm":
        o = ops.rms_norm_quantize(s["x"], s["weight"], EPS, residual=s["residual"], fake_quant=True)
        out = {"values": o["fq"], "scale": o["scale"]}
        return out if s["residual"] is None else dict(out, residual=o["residual"])
    if s["op"] == "quantise":
        return {"values": ops.quantize_fp4(s["x"], s["fmt"], global_scale=s["x_global"], fake_quant=True)["fq"]}
    w = ops.Fp4Tensor(s["w_codes"], s["w_scales"], s["N"], s["K"], s["fmt"], s["w_global"])
    act = ops.ACT_GELU if s["gelu"] else ops.ACT_NONE
    if s["op"] == "product":
        a = ops.Fp4Tensor(s["x_codes"], s["x_scales"], s["M"], s["K"], s["fmt"])
        return {"y": ops.gemm_fp4(a, w, bias=s["bias"], residual=s["residual"], activation=act, out_dtype=s["dtype"])}
    return {"y": ops.linear_fp4(s["x"], w, bias=s["bias"], residual=s["residual"], activation=act, out_dtype=s["dtype"])}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- inputs -----------------------------------------------------------------------------------------

def _activation(rows, K, gen, dtype):
    """N(0, 1) with one channel in a hundred twenty times as large, the outlier channels of transformer activations."""
    x = torch.randn((rows, K), generator=gen, device="cuda")
    x *= 1.0 + 19.0 * (torch.rand((K,), generator=gen, device="cuda") < 0.01)
    return x.to(dtype)


def _global(x):
    """The power of two that brings the largest block scale of x into (224, 448], as a layer keeps it."""
    return 2.0 ** math.ceil(math.log2(max(float(x.abs().max()), 1e-30) / (6.0 * 448.0)))


def _inputs(case, seed):
    """The float inputs of a case: what both prepare and exact start from."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    M, K, dt = case["M"], case["K"], DTYPE[case["dtype"]]
    s = {"x": _activation(M, K, gen, dt)}
    if case["op"] == "norm":
        s["weight"] = (1.0 + 0.2 * torch.randn((K,), generator=gen, device="cuda")).to(dt)
        s["residual"] = _activation(M, K, gen, dt) if case["residual"] else None
    elif case["op"] == "quantise":
        s["x_global"] = _global(s["x"]) if case["global_scale"] else 1.0
    else:
        N = case["N"]
        s["w"] = 0.02 * torch.randn((N, K), generator=gen, device="cuda")
        s["w_global"] = _global(s["w"]) if case["fmt"] == "nvfp4" else 1.0
        s["bias"] = (0.1 * torch.randn((N,), generator=gen, device="cuda")).to(dt) if case["bias"] else None
        s["residual"] = _activation(M, N, gen, dt) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s.update(op=case["op"], M=case["M"], K=case["K"], dtype=DTYPE[case["dtype"]], fmt=case.get("fmt"), gelu=case.get("gelu"), N=case.get("N"))
    if case["op"] in ("product", "linear"):
        v, scale, _ = _quantise_plain(s["w"], case["fmt"], s["w_global"])
        s["w_codes"], s["w_scales"] = _store(v, scale, case["fmt"], case["K"])
        del s["w"]
    if case["op"] == "product":
        v, scale, _ = _quantise_plain(s["x"], case["fmt"], 1.0)
        s["x_codes"], s["x_scales"] = _store(v, scale, case["fmt"], case["K"])
        del s["x"]
    return s


def work(case):
    M, K, e = case["M"], case["K"], SIZE[case["dtype"]]
    if case["op"] == "norm":                       # x, residual, weight in; residual, codes, values, scales out
        r = 2 if case["residual"] else 0
        return {"bytes": M * K * (e * (2 + r) + 1) + K * e + 4 * M, "flops": 10 * M * K}
    four = 0.5 + 1.0 / BLOCK[case["fmt"]]          # bytes of an element with its share of a scale
    if case["op"] == "quantise":                   # x in; codes, scales, values out
        return {"bytes": M * K * (2 * e + four), "flops": 5 * M * K}
    N = case["N"]
    x = M * K * (four if case["op"] == "product" else e)
    tail = e * ((N if case["bias"] else 0) + M * N * (2 if case["residual"] else 1))
    return {"bytes": x + N * K * four + tail, "flops": 2 * M * N * K}


# ---- the definitions in 64 bits ---------------------------------------------------------------------

def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3_64(v):
    """Nearest e4m3 value (ties to the even code) of 0 <= v <= 448: four significant bits, spacing 2^-9 at least."""
    step = _pow2_64(torch.frexp(v.clamp(min=2.0 ** -20)).exponent.clamp(min=-5) - 4)
    return torch.round(v / step) * step


def _four_bits_64(x, fmt, g):
    """The values that a 4-bit operand with the global scale g stands for, [rows, K] in 64 bits."""
    rows, K = x.shape
    b = BLOCK[fmt]
    nb = -(-K // b)
    z = torch.zeros((rows, nb * b), dtype=torch.float64, device=x.device)
    z[:, :K] = x.double()
    z = z.view(rows, nb, b)
    top = z.abs().max(-1, keepdim=True).values
    if fmt == "mxfp4":
        block = _pow2_64(torch.frexp(top.clamp(min=2.0 ** -125)).exponent - 3)
    else:
        block = _e4m3_64((top / (6.0 * g)).clamp(max=448.0)).clamp(min=2.0 ** -9)
    a = (z / (block * g)).abs()
    q = torch.zeros_like(a)
    # borders between neighbouring magnitudes; a value on one goes to the even code
    for border, odd, jump in ((0.25, False, 0.5), (0.75, True, 0.5), (1.25, False, 0.5), (1.75, True, 0.5), (2.5, False, 1.0), (3.5, True, 1.0), (5.0, False, 2.0)):
        q += jump * ((a >= border) if odd else (a > border))
    return (q * z.sign() * (block * g)).view(rows, nb * b)[:, :K]


def exact(case, seed):
    s = _inputs(case, seed)
    x = s["x"]
    if case["op"] == "norm":
        h = x.double() if s["residual"] is None else (x.float() + s["residual"].float()).to(x.dtype).double()
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / case["K"] + EPS) * s["weight"].double()
        scale = y.abs().max(-1, keepdim=True).values.clamp(min=1e-5) / 127.0
        out = {"values": torch.round(y / scale) * scale, "scale": scale[:, 0]}
        return out if s["residual"] is None else dict(out, residual=x.double() + s["residual"].double())
    if case["op"] == "quantise":
        return {"values": _four_bits_64(x, case["fmt"], s["x_global"])}
    y = _four_bits_64(x, case["fmt"], 1.0) @ _four_bits_64(s["w"], case["fmt"], s["w_global"]).T
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["gelu"]:
        y = y * torch.special.ndtr(y)
    return {"y": y if s["residual"] is None else y + s["residual"].double()}

"""Microscaled 4-bit floating point on the GPU: the quantizer bit for bit against the 64-bit oracle, the product
exactly where its sums are exact, and within derived bounds elsewhere."""
import numpy as np
import pytest
import torch

from oracle import fp4 as F
from sam_quantization_b200 import _lib, ops

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp4", "nvfp4"]
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _values(M, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + 17 * M + K)
    x = torch.randn(M, K, generator=g) * torch.exp(2.0 * torch.randn(M, 1, generator=g))
    x = x * (1.0 + 19.0 * (torch.rand(K, generator=g) < 0.02))
    return x.to(dtype)


def _check_quantized(x, out, fmt, g=1.0):
    M, K = x.shape
    code, byte, value = F.quantize(x.double().cpu().numpy(), fmt, g)
    q = out["q"]
    assert (q.rows, q.K, q.fmt, q.global_scale) == (M, K, fmt, g)
    assert np.array_equal(q.codes.cpu().numpy(), F.pack_codes(code, q.codes.shape[1]))
    assert np.array_equal(q.scales.cpu().numpy(), F.tile_scales(byte, fmt, K))
    want = torch.from_numpy(value).to(x.dtype)
    assert torch.equal(torch.nan_to_num(out["fq"].cpu(), nan=-77.0), torch.nan_to_num(want, nan=-77.0))
    assert torch.equal(torch.nan_to_num(q.dequantize(x.dtype).cpu(), nan=-77.0), torch.nan_to_num(want, nan=-77.0))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 16), (3, 31), (5, 33), (128, 256), (129, 257), (130, 1282), (131, 1283), (40, 70), (7, 5120), (300, 64), (33, 1023)])
def test_quantizer_equals_the_oracle(cuda_device, fmt, dtype, M, K):
    x = _values(M, K, dtype)
    _check_quantized(x, ops.quantize_fp4(x.to(cuda_device), fmt, fake_quant=True), fmt)


@pytest.mark.parametrize("g", [2.0 ** -14, 0.5, 8.0])
def test_global_scale(cuda_device, g):
    x = _values(65, 200, torch.float32) * 0.02
    _check_quantized(x, ops.quantize_fp4(x.to(cuda_device), "nvfp4", global_scale=g, fake_quant=True), "nvfp4", g)


@pytest.mark.parametrize("fmt", FORMATS)
def test_borders_between_codes_and_scales(cuda_device, fmt):
    """Every border of a code and its neighbours in fp32, under scales of every mantissa; block maxima at and next to
    the borders of the scale."""
    rows = []
    for m in (8, 9, 10, 11, 12, 13, 14, 15):
        s = m / 8.0 if fmt == "nvfp4" else 2.0 ** (m - 10)
        for b in list(F.BORDERS) + [6.0, 0.5]:
            v = np.float32(b * s)
            rows.append([np.float32(6 * s), v, np.nextafter(v, np.float32(0)), np.nextafter(v, np.float32(99)), -v] + [0.0] * 11)
    mids = (F.E4M3[1:] + F.E4M3[:-1]) / 2 * 6
    for v in list(mids) + list(F.E4M3 * 6) + [2.0 ** i for i in range(-20, 20)]:
        v = np.float32(v)
        for t in (v, np.nextafter(v, np.float32(0)), np.nextafter(v, np.float32(1e9))):
            rows.append([t] + [0.3 * t, -0.7 * t] + [0.0] * 13)
    x = torch.tensor(np.array(rows, np.float32))
    x = torch.cat((x, x.flip(0)), 1)
    _check_quantized(x, ops.quantize_fp4(x.to(cuda_device), fmt, fake_quant=True), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_extreme_values(cuda_device, fmt):
    x = torch.zeros(9, 70)
    x[1] = 3e38 * torch.linspace(-1, 1, 70)
    x[2] = 1e-38 * torch.linspace(-1, 1, 70)
    x[3] = 1e-44
    x[4, 3] = float("nan")
    x[5, 40] = float("inf")
    x[6, 69] = -float("inf")
    x[7] = torch.linspace(-1e-3, 1e-3, 70)
    x[8] = -0.0
    _check_quantized(x, ops.quantize_fp4(x.to(cuda_device), fmt, fake_quant=True), fmt)
    x16 = x.clamp(-65504, 65504)
    x16[4, 3], x16[5, 40] = float("nan"), float("inf")
    x16 = x16.half()
    _check_quantized(x16, ops.quantize_fp4(x16.to(cuda_device), fmt, fake_quant=True), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K,pitch,offset", [(256, 264, 0), (256, 259, 0), (250, 300, 3)])
def test_rows_with_a_pitch(cuda_device, fmt, K, pitch, offset):
    x = _values(20, pitch, torch.bfloat16).to(cuda_device)[:, offset:offset + K]
    _check_quantized(x.cpu(), ops.quantize_fp4(x, fmt, fake_quant=True), fmt)
    x = _values(12, K, torch.float16).to(cuda_device)
    out = ops.quantize_fp4(x.view(3, 4, K), fmt, fake_quant=True)
    assert out["fq"].shape == (3, 4, K)
    _check_quantized(x.cpu(), {"q": out["q"], "fq": out["fq"].view(12, K)}, fmt)


def test_no_rows(cuda_device):
    x = torch.empty(0, 64, dtype=torch.float16, device=cuda_device)
    w = ops.quantize_fp4(_values(24, 64, torch.float16).to(cuda_device))["q"]
    out = ops.quantize_fp4(x, fake_quant=True)
    assert out["fq"].shape == (0, 64)
    assert ops.gemm_fp4(out["q"], w).shape == (0, 24) and ops.linear_fp4(x, w).shape == (0, 24)


# ---- the product ----------------------------------------------------------------------------------------

def _exact_operand(rows, K, fmt, dev, seed):
    """Random codes under scales of two neighbouring exponents (and e4m3 mantissas): every product and partial sum is a
    multiple of 2^-6 below 2^17, exact in fp32 in any order."""
    rng = np.random.default_rng(seed)
    code = rng.integers(0, 16, (rows, K)).astype(np.uint8)
    nb = -(-K // F.BLOCK[fmt])
    byte = (rng.integers(126, 128, (rows, nb)) if fmt == "mxfp4" else rng.integers(0x30, 0x3B, (rows, nb)) & 0xFE).astype(np.uint8)
    pitch = (K + 31) // 32 * 16
    q = ops.Fp4Tensor(torch.from_numpy(F.pack_codes(code, pitch)).to(dev), torch.from_numpy(F.tile_scales(byte, fmt, K)).to(dev), rows, K, fmt)
    value = F.code_value(code) * np.repeat(F.scale_value(byte, fmt), F.BLOCK[fmt], 1)[:, :K]
    return q, value


SHAPES = [(1, 1, 1), (1, 8, 64), (3, 130, 31), (1, 5120, 1280), (128, 128, 256), (129, 257, 300), (200, 40, 1283), (64, 1001, 512), (16, 300, 2048),
          (17, 65, 96), (40, 200, 4100), (260, 520, 768), (1000, 384, 200), (300, 1280, 5120), (1, 20000, 300), (200, 7000, 256), (24, 2304, 768), (2600, 1300, 600), (8200, 257, 1283), (290, 8210, 300), (4096, 2304, 768),
          # enough tiles for the pair kernel, A resident and not
          (40000, 20, 100), (39990, 130, 1300), (5000, 1301, 1280), (5001, 1300, 1281), (300, 20000, 520), (20000, 384, 2600), (700, 9000, 3)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_product_is_exact_where_its_sums_are(cuda_device, fmt, M, N, K):
    a, av = _exact_operand(M, K, fmt, cuda_device, M + K)
    w, wv = _exact_operand(N, K, fmt, cuda_device, N + K + 1)
    y = ops.gemm_fp4(a, w, out_dtype=torch.float32)
    torch.cuda.synchronize()
    ops.check_status()
    assert np.array_equal(y.cpu().numpy().astype(np.float64), av @ wv.T)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 300, 1280), (5, 72, 100), (40, 1001, 2000), (130, 257, 1283), (600, 640, 512), (2050, 1096, 300), (5050, 1096, 300), (5050, 1101, 1400)])
@pytest.mark.parametrize("bias,gelu,residual", [(True, False, False), (True, True, False), (False, False, True), (True, True, True)])
def test_epilogue(cuda_device, fmt, dtype, M, N, K, bias, gelu, residual):
    """Exact sums, so only the epilogue rounds: alpha and bias in one fused step (u), GELU (3e-7 absolute and 2e-5
    relative, csrc/gemm_common.cuh), the residual's addition (u) and the rounding to the output type."""
    a, av = _exact_operand(M, K, fmt, cuda_device, 1)
    w, wv = _exact_operand(N, K, fmt, cuda_device, 2)
    a.global_scale, w.global_scale = 0.25, 2.0 ** -6
    g = torch.Generator().manual_seed(5)
    b = torch.randn(N, generator=g).to(dtype) if bias else None
    r = torch.randn(M, N, generator=g).to(dtype) if residual else None
    y = ops.gemm_fp4(a, w, bias=None if b is None else b.to(cuda_device), residual=None if r is None else r.to(cuda_device),
                     activation=ops.ACT_GELU if gelu else ops.ACT_NONE, out_dtype=dtype)
    ops.check_status()
    z = (av @ wv.T) * 2.0 ** -8
    if b is not None:
        z = z + b.double().numpy()
    u = 2.0 ** -24
    tol = u * np.abs(z)
    if gelu:
        tol = tol * 1.2 + 3e-7 + 2e-5 * np.abs(z)                      # |gelu'| < 1.13
        z = F.gelu(z)
    if r is not None:
        z = z + r.double().numpy()
        tol = tol + u * np.abs(z)
    tol = tol + HALF[dtype] * (np.abs(z) + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert np.all(np.abs(y.double().cpu().numpy() - z) <= tol)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 640, 1280), (37, 200, 1283), (300, 300, 5120)])
def test_product_of_quantized_data(cuda_device, fmt, M, N, K):
    """Scales over many exponents.  fp32 accumulation of at most K terms, each addition off by at most a step of the sum
    of magnitudes S: K * 2^-23 * S."""
    x = _values(M, K, torch.bfloat16)
    wt = (torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02)
    g = ops.fp4_global_scale(float(wt.abs().max())) if fmt == "nvfp4" else 1.0
    w = ops.quantize_fp4(wt.to(cuda_device), fmt, global_scale=g)["q"]
    y = ops.gemm_fp4(ops.quantize_fp4(x.to(cuda_device), fmt)["q"], w, out_dtype=torch.float32)
    ops.check_status()
    av, wv = F.quantize(x.double().numpy(), fmt)[2], F.quantize(wt.double().numpy(), fmt, g)[2]
    tol = K * 2.0 ** -23 * (np.abs(av) @ np.abs(wv).T)
    assert np.all(np.abs(y.double().cpu().numpy() - av @ wv.T) <= tol + 1e-30)
    # and the layer in one call is the two calls
    z = ops.linear_fp4(x.to(cuda_device), w, out_dtype=torch.float32)
    assert np.all(np.abs(z.double().cpu().numpy() - av @ wv.T) <= tol + 1e-30)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 640, 1280), (3, 131, 33), (8, 300, 5120), (9, 1000, 300), (17, 200, 1283), (32, 257, 2048)])
def test_one_kernel_layer_equals_its_two_halves(cuda_device, fmt, dtype, M, N, K):
    """linear_fp4 of at most 32 rows quantizes inside the product.  Exactly representable data: the layer's output is the
    quantizer's values times the weight, exactly, in any order of summation."""
    rng = np.random.default_rng(M + N + K)
    w, wv = _exact_operand(N, K, fmt, cuda_device, 7)
    # code values under block scales 2^-1 and 2^0, each block with a 6 so that quantization gives the values back
    b = F.BLOCK[fmt]
    nb = -(-K // b)
    v = F.code_value(rng.integers(0, 16, (M, nb, b)))
    v[:, :, 0] = 6.0
    xv = (v * rng.choice([0.5, 1.0], (M, nb, 1))).reshape(M, nb * b)[:, :K]
    x = torch.from_numpy(xv).to(dtype).to(cuda_device)
    g = torch.Generator().manual_seed(5)
    bias, res = torch.randn(N, generator=g).to(dtype), torch.randn(M, N, generator=g).to(dtype)
    y = ops.linear_fp4(x, w, bias=bias.to(cuda_device), residual=res.to(cuda_device))
    ops.check_status()
    z = xv @ wv.T + bias.double().numpy()
    u = 2.0 ** -24
    tol = u * np.abs(z)
    z = z + res.double().numpy()
    tol = tol + u * np.abs(z)
    tol = tol + HALF[dtype] * (np.abs(z) + tol)
    finite = np.abs(z) < (60000 if dtype == torch.float16 else 1e30)
    assert np.all(np.abs(y.double().cpu().numpy() - z)[finite] <= tol[finite])
    # a pitch, an offset that no vector may start at, and a leading shape
    wide = torch.randn(M, K + 5, device=cuda_device).to(dtype)
    wide[:, 3:K + 3] = x
    assert _same_bytes(ops.linear_fp4(wide[:, 3:K + 3], w, bias=bias.to(cuda_device), residual=res.to(cuda_device)), y)
    assert ops.linear_fp4(x.view(M, 1, K), w).shape == (M, 1, N)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,N,K", [(1, 700, 10240), (9, 5003, 5130), (16, 20000, 5120), (24, 2700, 4099), (32, 10240, 5120), (32, 640, 1290)])
def test_layer_of_few_rows_is_the_same_with_and_without_a_workspace(cuda_device, fmt, M, N, K):
    """Given a workspace, the library may quantize first; the sums are the same, in the same order.  Clusters of every size."""
    lib, g = _lib.load(), torch.Generator().manual_seed(M + N)
    x = torch.randn(M, K, generator=g).to(torch.bfloat16).to(cuda_device)
    w = ops.quantize_fp4(torch.randn(N, K, generator=g).to(torch.bfloat16).to(cuda_device), fmt)["q"]
    y = ops.linear_fp4(x, w)
    two = ops.gemm_fp4(ops.quantize_fp4(x, fmt)["q"], w, out_dtype=torch.bfloat16)
    one = torch.empty_like(y)
    rc = lib.samq_linear_fp4(x.data_ptr(), _lib.BF16, K, w.codes.data_ptr(), w.codes.stride(0), w.scales.data_ptr(), M, N, K, ops.FP4_FORMATS[fmt],
                             w.global_scale, None, None, 0, 0, one.data_ptr(), _lib.BF16, N, None, 0, None, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    ops.check_status()
    assert _same_bytes(y, two) and _same_bytes(one, two)


def _same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M", [1, 33, 200, 40001])
def test_rows_that_are_not_finite_stay_apart(cuda_device, fmt, M):
    x = _values(M, 300, torch.float16)
    x[M // 2, 299] = float("nan")
    w, wv = _exact_operand(50, 300, fmt, cuda_device, 3)
    for act in (ops.ACT_NONE, ops.ACT_GELU):
        y = ops.linear_fp4(x.to(cuda_device), w, activation=act)
        ops.check_status()
        bad = ~x.isfinite().all(1).to(cuda_device)                       # (a value of the others can be an fp16 infinity too)
        assert bad[M // 2] and torch.equal(y.isnan().all(1), bad) and torch.equal(y.isnan().any(1), bad)


@pytest.mark.parametrize("K", [200, 1500])
@pytest.mark.parametrize("N,res_pitch", [(1096, 1101), (1101, 1112), (1101, 1101), (1096, 1104)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_outputs_and_residuals_with_and_without_a_tensor_map(cuda_device, dtype, N, res_pitch, K):
    """Rows of 16 bytes go by TMA, others element by element, the two of a call independently of one another."""
    M = 5050
    a, av = _exact_operand(M, K, "nvfp4", cuda_device, 1)
    w, wv = _exact_operand(N, K, "nvfp4", cuda_device, 2)
    w.global_scale = 2.0 ** -8
    res = torch.randn(M, res_pitch, generator=torch.Generator().manual_seed(3)).to(dtype).to(cuda_device)[:, :N]
    y = ops.gemm_fp4(a, w, residual=res, out_dtype=dtype)
    ops.check_status()
    z = av @ wv.T * 2.0 ** -8 + res.double().cpu().numpy()
    tol = 2.0 ** -24 * np.abs(z)
    tol = tol + HALF[dtype] * (np.abs(z) + tol) + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert np.all(np.abs(y.double().cpu().numpy() - z) <= tol)


@pytest.mark.parametrize("M", [3, 200, 700, 20001])
def test_strided_outputs_and_operands(cuda_device, M):
    a, av = _exact_operand(M, 320, "nvfp4", cuda_device, 1)
    w, wv = _exact_operand(130, 320, "nvfp4", cuda_device, 2)
    wide = torch.zeros(M, 192, dtype=torch.uint8, device=cuda_device)
    wide[:, :160] = a.codes
    wide[:, 160:] = 255                                                  # never read: behind K
    a2 = ops.Fp4Tensor(wide, a.scales, M, 320, "nvfp4")
    assert np.array_equal(ops.gemm_fp4(a2, w, out_dtype=torch.float32).double().cpu().numpy(), av @ wv.T)
    res = torch.randn(M, 140, device=cuda_device)[:, 3:133]              # a residual of unaligned rows
    y = ops.gemm_fp4(a, w, residual=res, out_dtype=torch.float32)
    assert np.array_equal(y.double().cpu().numpy(), np.float32(np.float32(av @ wv.T) + res.cpu().numpy()).astype(np.float64))
    out = torch.full((M + 2, 130), 9.0, dtype=torch.float32, device=cuda_device)
    ops.gemm_fp4(a, w, out_dtype=torch.float32, out=out[1:M + 1])
    assert (out[0] == 9).all() and (out[-1] == 9).all()                  # rows before and behind stay
    assert np.array_equal(out[1:M + 1].double().cpu().numpy(), av @ wv.T)


def test_refusals(cuda_device):
    a, _ = _exact_operand(4, 64, "nvfp4", cuda_device, 1)
    w, _ = _exact_operand(8, 64, "nvfp4", cuda_device, 2)
    m, _ = _exact_operand(8, 64, "mxfp4", cuda_device, 2)
    k, _ = _exact_operand(8, 96, "nvfp4", cuda_device, 2)
    x = torch.zeros(4, 64, dtype=torch.float16, device=cuda_device)
    for bad in (lambda: ops.gemm_fp4(a, m), lambda: ops.gemm_fp4(a, k), lambda: ops.linear_fp4(x, k), lambda: ops.quantize_fp4(x, "int4"),
                lambda: ops.gemm_fp4(a, w, bias=torch.zeros(7, dtype=torch.float16, device=cuda_device)),
                lambda: ops.gemm_fp4(a, w, residual=x), lambda: ops.gemm_fp4(a, w, out=x)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.gemm_fp4(a, w, out_dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.gemm_fp4(a, w, residual=torch.zeros(4, 8, device=cuda_device))
    with pytest.raises(RuntimeError, match="global_scale"):
        ops.quantize_fp4(x, "nvfp4", global_scale=3.0)
    with pytest.raises(RuntimeError, match="mxfp4"):
        ops.quantize_fp4(x, "mxfp4", global_scale=2.0)


def _same(a, b):
    """Bit for bit (a row of these values can hold an fp16 infinity, and is then NaN on both sides)."""
    return torch.equal(a.view(torch.int16), b.view(torch.int16))


@pytest.mark.parametrize("M", [2, 150, 20000])
def test_captured_replayed_and_on_two_streams(cuda_device, M):
    x = _values(M, 640, torch.float16).to(cuda_device)
    x2 = _values(M, 640, torch.float16, seed=4).to(cuda_device)
    w = ops.quantize_fp4((torch.randn(300, 640, generator=torch.Generator().manual_seed(1)) * 0.02).to(cuda_device))["q"]
    want, want2 = ops.linear_fp4(x, w), ops.linear_fp4(x2, w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):                                                   # two calls at once
        with torch.cuda.stream(side):
            y2 = ops.linear_fp4(x2, w)
        y = ops.linear_fp4(x, w)
    torch.cuda.current_stream().wait_stream(side)
    assert _same(y, want) and _same(y2, want2)
    graphs = []
    for src in (x, x2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.linear_fp4(src, w)
        graphs.append((graph, out))
    for _ in range(3):
        for graph, _ in graphs:
            graph.replay()
    assert _same(graphs[0][1], want) and _same(graphs[1][1], want2)
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("g", [2.0 ** -64, 2.0 ** -40, 2.0 ** -14, 0.5, 2.0 ** 20, 2.0 ** 64])
def test_extreme_values_under_a_global_scale(cuda_device, dtype, g):
    """Blocks far beyond the largest scale saturate (and stay finite), blocks far below the smallest round to zero."""
    top = float(torch.finfo(dtype).max)
    x = torch.zeros(12, 70)
    for i, size in enumerate((top, 3e38, 3e34, 1e30, 1e20, 1e-20, 1e-38, 1e-44)):
        x[i] = min(size, top) * torch.linspace(-1, 1, 70)
    x[8] = min(3e38, top) * torch.logspace(0, -70, 70) * (1 - 2 * (torch.arange(70) % 2))      # every magnitude beside the largest
    x[9] = g * torch.linspace(-3000, 3000, 70)
    x[10, 3], x[10, 60] = float("nan"), 1e30
    x[11, 40], x[11, 3] = -float("inf"), -1e30
    x = x.clamp(-top, top) if dtype == torch.float16 else x
    x[10, 3], x[11, 40] = float("nan"), -float("inf")
    x = x.to(dtype)
    _check_quantized(x, ops.quantize_fp4(x.to(cuda_device), "nvfp4", global_scale=g, fake_quant=True), "nvfp4", g)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [-20, -13, 9, 30])
@pytest.mark.parametrize("M,N,K", [(1, 300, 1283), (8, 264, 300), (32, 640, 5120), (40, 200, 1280), (300, 130, 520), (4000, 1300, 300)])
def test_layer_under_an_activation_scale(cuda_device, dtype, k, M, N, K):
    """Activations of another power of two under a scale that follows them: the same codes, so the same output times that
    power, bit for bit.  (K = 5120 and 32 rows quantize first, since the wrapper gives a workspace.)"""
    x = _values(M, K, dtype).clamp(-2000, 2000).to(cuda_device)
    w = ops.quantize_fp4((torch.randn(N, K, generator=torch.Generator().manual_seed(1)) * 0.02).to(cuda_device), global_scale=2.0 ** -14)["q"]
    y = ops.linear_fp4(x, w, out_dtype=torch.float32)
    z = ops.linear_fp4(x * 2.0 ** k, w, out_dtype=torch.float32, x_global_scale=2.0 ** k)
    assert torch.equal(z, y * 2.0 ** k)
    # output of the activation's type: one kernel up to 32 rows
    b = (torch.randn(N, generator=torch.Generator().manual_seed(2)) * 2.0 ** k).to(dtype).to(cuda_device)
    z = ops.linear_fp4(x * 2.0 ** k, w, bias=b, x_global_scale=2.0 ** k)
    a = ops.quantize_fp4(x * 2.0 ** k, "nvfp4", global_scale=2.0 ** k)["q"]
    assert _same_bytes(z, ops.gemm_fp4(a, w, bias=b, out_dtype=dtype))
    ops.check_status()


@pytest.mark.parametrize("M", [1, 8, 40, 200])
@pytest.mark.parametrize("size", [1e-4, 1e4])
def test_small_and_large_activations(cuda_device, M, size):
    """Against the float product.  An element is off by at most half of the largest spacing (2, from 4 on) times its block's
    scale, which is at most max / 6 * (1 + 2^-4) (and a block's largest, up to 6 / (1 - 2^-4) scales, by 0.4 of them)."""
    K, N = 640, 96
    x = (torch.randn(M, K, generator=torch.Generator().manual_seed(M)) * size).to(torch.bfloat16).to(cuda_device)
    w, wv = _exact_operand(N, K, "nvfp4", cuda_device, 3)
    g = ops.fp4_global_scale(float(x.abs().max()))
    xv = x.double().cpu().numpy()
    top = np.repeat(np.abs(xv).reshape(M, K // 16, 16).max(-1), 16, 1) * (1.0625 / 6)
    for out_dtype in (torch.bfloat16, torch.float32):                      # one kernel and two, for few rows
        y = ops.linear_fp4(x, w, out_dtype=out_dtype, x_global_scale=g).double().cpu().numpy()
        bound = top @ np.abs(wv).T
        want = xv @ wv.T
        assert np.all(np.abs(y - want) <= bound + (HALF[out_dtype] + K * 2.0 ** -23) * (np.abs(xv) @ np.abs(wv).T + bound))
        assert np.corrcoef(y.ravel(), want.ravel())[0, 1] > 0.98
    with pytest.raises(RuntimeError, match="global_scale"):
        ops.linear_fp4(x, w, x_global_scale=3.0)
    m, _ = _exact_operand(N, K, "mxfp4", cuda_device, 3)
    with pytest.raises(RuntimeError, match="mxfp4"):
        ops.linear_fp4(x, m, x_global_scale=2.0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("g", [1.0, 0.25, 2.0 ** 20])
def test_dequantized_values_are_what_the_product_multiplies(cuda_device, fmt, g):
    a, av = _exact_operand(70, 45, fmt, cuda_device, 1)
    a.global_scale = g
    eye = ops.quantize_fp4(6 * torch.eye(45, device=cuda_device), fmt)["q"]              # blocks of a six: scale 1
    y = ops.gemm_fp4(a, eye, out_dtype=torch.float32)
    assert np.array_equal(a.dequantize().double().cpu().numpy(), av * g) and torch.equal(a.dequantize() * 6, y)
    a.global_scale = 0.3                                                                 # any float in a product
    assert torch.allclose(a.dequantize() * 6, ops.gemm_fp4(a, eye, out_dtype=torch.float32), rtol=4 * 2.0 ** -24, atol=0)


@pytest.mark.parametrize("M,N,K,out_dtype,kernels", [(1, 640, 1280, None, 1), (32, 640, 1280, None, 1), (32, 20000, 5120, None, 2), (1, 20000, 10240, None, 2),
                                                     (32, 640, 5120, None, 1), (33, 640, 1280, None, 2), (1, 640, 1280, torch.float32, 2)])
def test_launches_of_a_layer_are_counted(cuda_device, M, N, K, out_dtype, kernels):
    """The count is the library's own choice of one or two kernels: the rule that its dispatch goes by."""
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).to(torch.bfloat16).to(cuda_device)
    w = ops.quantize_fp4(torch.randn(N, K, device=cuda_device) * 0.02)["q"]
    ops.reset_counters()
    ops.linear_fp4(x, w, out_dtype=out_dtype)
    assert ops.launch_count() == kernels
    ops.check_status()


@pytest.mark.parametrize("e", [-64, 63])
def test_global_scales_at_their_ends(cuda_device, e):
    """The product of two scales 2^64 is beyond fp32 and refused; 2^-64 and 2^-64 make a subnormal alpha, which is exact."""
    a, av = _exact_operand(5, 100, "nvfp4", cuda_device, 1)
    w, wv = _exact_operand(30, 100, "nvfp4", cuda_device, 2)
    a.global_scale, w.global_scale = 2.0 ** e, 2.0 ** e
    y = ops.gemm_fp4(a, w, out_dtype=torch.float32)
    want = (av @ wv.T) * 2.0 ** (2 * e)
    with np.errstate(over="ignore"):
        assert np.array_equal(y.cpu().numpy(), want.astype(np.float32))
    a.global_scale = w.global_scale = 2.0 ** 64
    with pytest.raises(RuntimeError, match="alpha"):
        ops.gemm_fp4(a, w, out_dtype=torch.float32)
    with pytest.raises(RuntimeError, match="alpha"):
        ops.linear_fp4(torch.ones(5, 100, device=cuda_device), w, x_global_scale=2.0 ** 64)


def test_kernel_timing_tells_operations_from_bytes(cuda_device):
    M, N, K = 40, 64, 96
    a, _ = _exact_operand(M, K, "nvfp4", cuda_device, 1)
    w, _ = _exact_operand(N, K, "nvfp4", cuda_device, 2)
    x = torch.zeros(M, K, dtype=torch.float16, device=cuda_device)
    ops.enable_kernel_timing(True)
    try:
        ops.gemm_fp4(a, w)
        ops.linear_fp4(x, w)
        ops.quantize_fp4(x)
        ops.rms_norm_quantize(x, x[0])
        got = ops.kernel_timing_summary()
    finally:
        ops.enable_kernel_timing(False)
    for kind in ("gemm_fp4", "linear_fp4"):
        assert (got[kind]["ops"], got[kind]["bytes"], got[kind]["launches"]) == (2.0 * M * N * K, 0.0, 1)
    assert got["quant_fp4"]["ops"] == got["rms_norm_quant"]["ops"] == 0.0
    assert got["quant_fp4"]["bytes"] == M * K * 2 + M * K // 2 + 128 * 16 and got["rms_norm_quant"]["bytes"] == M * K * 3 + 4 * M

"""RMS norm with an 8-bit output (``ops.rms_norm_quantize``) against the definition in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32).  The sum of K squares: at most 40 fused multiply-adds a thread, 5
levels of the warp and 32 warps, all terms positive: 77 u relative, 38.5 u after the root.  rsqrtf 4 u, 1/K and the
fused multiply-add 2 u, two products 2 u, the division by q_max 1 u: the scale is within 50 u.  A quotient y / s adds the
same for y and 2 u: |y / s| <= q_max, so it is within 127 * 100 u of the exact one, and a code within half a step more."""
import numpy as np
import pytest
import torch

from oracle import fp4 as F
from sam_quantization_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def _inputs(M, K, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + 131 * M + K)
    x = torch.randn(M, K, generator=g) * (1.0 + 19.0 * (torch.rand(K, generator=g) < 0.02))
    r = torch.randn(M, K, generator=g) * 3
    w = 1.0 + 0.3 * torch.randn(K, generator=g)
    return x.to(dtype).to(dev), r.to(dtype).to(dev), w.to(dtype).to(dev)


def _check(out, h, w, n_bits=8, eps=EPS):
    """``out`` of the rows ``h`` (the sum, in the tensor dtype) against the definition."""
    qmax = 2.0 ** (n_bits - 1) - 1
    quot, s = F.rms_norm(h.double().cpu().numpy(), w.double().cpu().numpy(), eps, qmax)
    got = out["scale"].double().cpu().numpy()
    assert np.all(np.abs(got - s) <= 50 * U * s)
    q = out["q"].cpu().numpy().astype(np.float64)
    assert np.abs(q).max() <= qmax
    assert np.all(np.abs(q - quot) <= 0.5 + qmax * 100 * U)
    if "fq" in out:                                        # exactly the codes times the scale, rounded once
        assert torch.equal(out["fq"], (out["q"].float() * out["scale"][:, None]).to(out["fq"].dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 1280), (3, 7), (5, 1023), (33, 1280), (17, 2048), (9, 4096), (3, 5120), (70, 96), (2, 8200), (65, 1281), (67, 1282), (130, 85), (40, 20), (19, 5119), (9, 8191), (2, 20481), (3, 31), (11, 12), (10, 3), (6, 257), (7, 515), (5, 4099), (3, 16383),
                                 (2, 20488), (1, 32767), (2, 32768)])
def test_matches_the_definition(cuda_device, dtype, M, K):
    x, r, w = _inputs(M, K, dtype, cuda_device)
    out = ops.rms_norm_quantize(x, w, EPS, fake_quant=True)
    assert out["q"].shape == (M, K) and out["q"].dtype == torch.int8 and "residual" not in out
    _check(out, x, w)
    out = ops.rms_norm_quantize(x, w, EPS, residual=r, fake_quant=True)
    h = (x.float() + r.float()).to(dtype)                  # one rounding of an exact or fp32 sum: bit for bit
    assert torch.equal(out["residual"], h)
    _check(out, h, w)


def test_small_batches_and_bits(cuda_device):
    x, r, w = _inputs(6, 640, torch.bfloat16, cuda_device)
    for n_bits in (2, 4, 7):
        _check(ops.rms_norm_quantize(x, w, EPS, n_bits=n_bits), x, w, n_bits)
    out = ops.rms_norm_quantize(x.view(2, 3, 640), w, EPS, residual=r.view(2, 3, 640))
    assert out["q"].shape == (2, 3, 640) and out["scale"].shape == (2, 3) and out["residual"].shape == (2, 3, 640)
    out = ops.rms_norm_quantize(x[:0], w, EPS, residual=r[:0], fake_quant=True)
    assert out["q"].shape == (0, 640) and out["scale"].shape == (0,)
    out = ops.rms_norm_quantize(x, w, EPS, codes=False, fake_quant=True)
    assert "q" not in out and torch.equal(out["fq"], ops.rms_norm_quantize(x, w, EPS, fake_quant=True)["fq"])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("K,pitch,offset", [(1280, 1408, 0), (1280, 1283, 0), (1280, 1408, 3), (77, 90, 1), (77, 85, 0), (1281, 1289, 0), (1279, 1287, 0)])
def test_rows_with_a_pitch_equal_contiguous_rows(cuda_device, dtype, K, pitch, offset):
    x, r, w = _inputs(9, pitch, dtype, cuda_device)
    xs, rs, ws = x[:, offset:offset + K], r[:, offset:offset + K], w[offset:offset + K]
    dst = torch.full((9, pitch), 7.0, dtype=dtype, device=cuda_device)
    got = ops.rms_norm_quantize(xs, ws, EPS, residual=rs, residual_out=dst[:, offset:offset + K])
    h = (xs.float() + rs.float()).to(dtype)
    assert torch.equal(dst[:, offset:offset + K], h)
    keep = torch.ones(pitch, dtype=torch.bool)
    keep[offset:offset + K] = False
    assert torch.equal(dst[:, keep], torch.full_like(dst[:, keep], 7.0))         # what lies between the rows stays
    _check(got, h, ws)


def test_the_residual_stream_is_updated_in_place(cuda_device):
    x, r, w = _inputs(40, 1280, torch.bfloat16, cuda_device)
    want = ops.rms_norm_quantize(x, w, EPS, residual=r)
    stream = r.clone()
    got = ops.rms_norm_quantize(x, w, EPS, residual=stream, residual_out=stream)
    assert got["residual"] is stream and torch.equal(stream, want["residual"]) and torch.equal(got["q"], want["q"])
    xin = x.clone()
    ops.rms_norm_quantize(xin, w, EPS, residual=r, residual_out=xin)
    assert torch.equal(xin, want["residual"])


def test_rows_of_zeros_and_rows_that_are_not_finite(cuda_device):
    x, _, w = _inputs(6, 1280, torch.float16, cuda_device)
    x[1] = 0
    x[2, 5] = float("nan")
    x[3, 1279] = float("inf")
    out = ops.rms_norm_quantize(x, w, EPS, fake_quant=True)
    fine = [0, 1, 4, 5]
    _check({k: v[fine] for k, v in out.items()}, x[fine], w)
    assert abs(float(out["scale"][1]) - 1e-5 / 127) < 1e-5 / 127 * 4 * U and int(out["q"][1].abs().max()) == 0
    assert out["scale"][2:4].isnan().all() and int(out["q"][2:4].abs().max()) == 0 and out["fq"][2:4].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("K", [257, 1279])
def test_odd_widths_first_and_last_elements(cuda_device, dtype, K):
    """Of an odd number of columns one a row stands apart from the pairs: the first or the last, by turns."""
    x, r, w = _inputs(8, K, dtype, cuda_device)
    x[0, K - 1], x[1, 0], x[2, 0], x[3, K - 1] = 40.0, -40.0, 40.0, -40.0         # the row's scale comes from there
    x[4, K - 1] = float("nan")
    x[5, 0] = float("inf")
    out = ops.rms_norm_quantize(x, w, EPS, residual=r, fake_quant=True)
    h = (x.float() + r.float()).to(dtype)
    assert torch.equal(out["residual"][:4], h[:4]) and torch.equal(out["residual"][6:], h[6:])
    fine = [0, 1, 2, 3, 6, 7]
    _check({k: v[fine] for k, v in out.items()}, h[fine], w)
    assert out["scale"][4:6].isnan().all() and int(out["q"][4:6].abs().max()) == 0 and out["fq"][4:6].isnan().all()
    stream = r.clone()
    again = ops.rms_norm_quantize(x, w, EPS, residual=stream, residual_out=stream, fake_quant=True)
    assert torch.equal(again["q"], out["q"]) and torch.equal(stream[fine], h[fine])


def test_large_rows_of_fp32_do_not_overflow_early(cuda_device):
    """Squares of 1e18 sum to 1e39 only behind fp32's range: the row is reported as not finite, others stand."""
    x, _, w = _inputs(2, 512, torch.float32, cuda_device)
    x[0] *= 1e17
    out = ops.rms_norm_quantize(x, w, EPS)
    _check(out, x, w)


def test_refusals(cuda_device):
    x, r, w = _inputs(4, 64, torch.float16, cuda_device)
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, w[:63])
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, w, residual=r[:3])
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, w, residual=r.float())
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, w, residual_out=r)
    with pytest.raises(ValueError):
        ops.rms_norm_quantize(x, w, residual=r, residual_out=torch.empty(64, 4, dtype=x.dtype, device=cuda_device).t())
    with pytest.raises(TypeError):
        ops.rms_norm_quantize(x.to(torch.int32), w)
    with pytest.raises(RuntimeError, match="n_bits"):
        ops.rms_norm_quantize(x, w, n_bits=12)


def test_captured_and_on_another_stream(cuda_device):
    x, r, w = _inputs(50, 1280, torch.float16, cuda_device)
    want = ops.rms_norm_quantize(x, w, EPS, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.rms_norm_quantize(x, w, EPS, residual=r)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got["q"], want["q"]) and torch.equal(got["scale"], want["scale"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.rms_norm_quantize(x, w, EPS, residual=r)
    x2, _, _ = _inputs(50, 1280, torch.float16, cuda_device, seed=9)
    x.copy_(x2)
    graph.replay()
    again = ops.rms_norm_quantize(x2, w, EPS, residual=r)
    assert torch.equal(out["q"], again["q"]) and torch.equal(out["residual"], again["residual"])


def test_feeds_the_int8_product(cuda_device):
    """norm -> int8 linear: the codes and scales are what gemm_i8 takes."""
    x, r, w = _inputs(130, 1280, torch.float16, cuda_device)
    g = torch.Generator().manual_seed(3)
    lin = (torch.randn(256, 1280, generator=g) * 0.02).half().to(cuda_device)
    wq = ops.quantize_weight(lin)
    out = ops.rms_norm_quantize(x, w, EPS, residual=r)
    y = ops.gemm_i8(out["q"], wq["q"], out["scale"], wq["scale"], out_dtype=torch.float32)
    want = (out["q"].double() * out["scale"].double()[:, None]) @ (wq["q"].double() * wq["scale"].double()[:, None]).t()
    # exact integer sums, then two fp32 products and a conversion: 4 u relative
    assert ((y.double() - want).abs() <= 4 * U * want.abs() + 1e-30).all()
    ops.check_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [1, 96, 160, 1279, 1280, 2050, 8191, 20488])
@pytest.mark.parametrize("eps", [1e-6, 0.0, 1e-30])
def test_rows_whose_squares_leave_the_range(cuda_device, dtype, K, eps):
    """Finite rows whose squares overflow fp32, or underflow it under a small eps, beside ordinary ones."""
    x, r, w = _inputs(9, K, torch.float32, cuda_device)
    x /= x.abs().amax(1, keepdim=True)
    # tiny rows down to 1e-30: below, the elements of a bf16 or fp32 row lose bits of their own
    for i, size in enumerate((3e19, 1.0, 1e30, 3e38, 1e-25, 1e-30, 5.0, 1e19, 1e-19)):
        x[i] *= size
    x, w = x.to(dtype), w.to(dtype)
    out = ops.rms_norm_quantize(x, w, eps, fake_quant=True)
    _check(out, x, w, eps=eps)
    out = ops.rms_norm_quantize(torch.zeros_like(x), w, eps, residual=x, fake_quant=True)      # the residual stream is not scaled
    assert torch.equal(out["residual"], x)
    _check(out, x, w, eps=eps)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("K", [96, 257, 1280])
def test_rows_of_zeros_without_an_eps(cuda_device, dtype, K):
    x, r, w = _inputs(5, K, dtype, cuda_device)
    x[1], x[4] = 0, -0.0
    x[2, K - 1] = float("inf")
    x[3, 0] = float("nan")
    out = ops.rms_norm_quantize(x, w, 0.0, fake_quant=True)
    _check({k: v[:1] for k, v in out.items()}, x[:1], w, eps=0.0)
    for i in (1, 4):
        assert abs(float(out["scale"][i]) - 1e-5 / 127) < 1e-5 / 127 * 4 * U
        assert int(out["q"][i].abs().max()) == 0 and int(out["fq"][i].count_nonzero()) == 0
    assert out["scale"][2:4].isnan().all() and int(out["q"][2:4].abs().max()) == 0 and out["fq"][2:4].isnan().all()

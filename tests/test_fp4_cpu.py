"""The 4-bit format and the RMS norm without a GPU: the oracle against known values, host helpers, and every refusal
(argument checks answer before any device work)."""
import math
import os
import pickle
import re

import numpy as np
import pytest
import torch

from oracle import fp4 as F
from sam_quantization_b200 import _lib, ops
from sam_quantization_b200.RTN_quantization import FP4Linear
from tests.test_abi_cpu import built_library


def test_oracle_rounds_to_nearest_even_codes():
    x = np.zeros((1, 32))
    x[0, :16] = [0.25, 0.26, 0.75, 0.74, 1.25, 1.75, 2.5, 3.5, 5.0, 5.1, 7.9, -0.75, -0.0, 0.5, -6.0, 4.0]
    code, byte, value = F.quantize(x, "mxfp4")                          # largest 7.9 -> scale 2^0
    assert byte.tolist() == [[127]]
    assert value[0, :16].tolist() == [0, 0.5, 1, 0.5, 1, 2, 2, 4, 4, 6, 6, -1, 0, 0.5, -6, 4]
    assert code[0, 11] == 10 and code[0, 12] == 8
    code, byte, value = F.quantize(np.array([[6.0] + [1.0] * 15, [6 * 448.0 * 4] + [0.0] * 15]), "nvfp4")
    assert byte.tolist() == [[0x38], [0x7E]] and value[0, 0] == 6 and value[1, 0] == 6 * 448
    assert len(F.E4M3) == 127 and F.E4M3[0x7E] == 448 and F.E4M3[1] == 2.0 ** -9


def test_oracle_layout_places_every_scale_once():
    byte = np.arange(200 * 20).reshape(200, 20).astype(np.uint8)
    t = F.tile_scales(byte, "nvfp4", 20 * 16)
    assert t.shape == (2, 8, 32, 4, 4) == ops.fp4_scale_shape("nvfp4", 200, 320)
    assert t[1, 2, 7, 1, 3] == byte[128 + 32 + 7, 11] and t[1, :, :, 3].sum() == 0
    assert ops.fp4_scale_shape("mxfp4", 129, 257) == (2, 4, 32, 4, 4)


@pytest.mark.parametrize("absmax", [1e-30, 0.02, 1.0, 2688.0, 2689.0, 1e30])
def test_global_scale_is_a_power_of_two_at_the_top_of_e4m3(absmax):
    g = ops.fp4_global_scale(absmax)
    assert math.frexp(g)[0] == 0.5
    if 2.0 ** -64 < g < 2.0 ** 64:
        assert 224.0 < absmax / (6.0 * g) <= 448.0
    assert ops.fp4_global_scale(0.0) == 1.0
    with pytest.raises(ValueError):
        ops.fp4_global_scale(float("inf"))


def test_scale_bytes_match_the_shape():
    built_library()
    lib = _lib.load()
    for fmt in ops.FP4_FORMATS:
        for rows, K in ((1, 1), (128, 256), (129, 257), (5, 5120)):
            assert lib.samq_fp4_scale_bytes(ops.FP4_FORMATS[fmt], rows, K) == math.prod(ops.fp4_scale_shape(fmt, rows, K))
    assert lib.samq_linear_fp4_workspace_bytes(_lib.FP4_NV, 33, 64) == 33 * 32 + 4 * 512
    assert lib.samq_linear_fp4_workspace_bytes(_lib.FP4_MX, 129, 257) == 129 * 144 + 2 * 4 * 512 and lib.samq_linear_fp4_workspace_bytes(9, 1, 1) == 0
    assert lib.samq_fp4_scale_bytes(7, 1, 1) == 0 and lib.samq_fp4_scale_bytes(0, 0, 16) == 0


def test_fp4_tensor_refuses_wrong_storage():
    codes, scales = torch.zeros((3, 16), dtype=torch.uint8), torch.zeros(ops.fp4_scale_shape("nvfp4", 3, 30), dtype=torch.uint8)
    ops.Fp4Tensor(codes, scales, 3, 30, "nvfp4")
    for bad in ((codes, scales, 3, 30, "int4"), (codes, scales, 4, 30, "nvfp4"), (codes, scales, 3, 34, "nvfp4"),
                (codes, scales, 3, 30, "mxfp4"), (codes, scales.view(-1), 3, 30, "nvfp4"), (codes.t(), scales, 16, 3, "nvfp4")):
        with pytest.raises(ValueError):
            ops.Fp4Tensor(*bad)
    with pytest.raises(TypeError):
        ops.Fp4Tensor(codes.char(), scales, 3, 30, "nvfp4")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    for call in (lambda: ops.quantize_fp4(x), lambda: ops.rms_norm_quantize(x, torch.ones(64))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def _calls(lib):
    one = 1 << 20                                       # an aligned address that no call may reach
    quant = dict(x=one, dtype=_lib.F16, M=4, K=64, ldx=64, fmt=_lib.FP4_NV, g=1.0, codes=one, ldq=32, scales=one, fq=None, stream=None)
    norm = dict(x=one, r=None, w=one, dtype=_lib.F16, M=4, K=64, ldx=64, ldr=0, eps=1e-6, n_bits=8, h=None, ldo=0, q=one, s=one, fq=None,
                stream=None)
    gemm = dict(A=one, lda=32, sa=one, W=one, ldw=32, sw=one, M=4, N=8, K=64, fmt=_lib.FP4_NV, alpha=1.0, bias=None, res=None, ldr=0,
                act=0, out=one, odt=_lib.F16, ldo=8, status=None, stream=None)
    lin = dict(x=one, dtype=_lib.F16, ldx=64, W=one, ldw=32, sw=one, M=4, N=8, K=64, fmt=_lib.FP4_NV, alpha=1.0, bias=None, res=None, ldr=0,
               act=0, out=one, odt=_lib.F16, ldo=8, ws=None, ws_bytes=0, status=None, stream=None)
    return {"linear": (lib.samq_linear_fp4, lin), "quant": (lib.samq_quant_fp4, quant), "norm": (lib.samq_rms_norm_quant_i8, norm), "gemm": (lib.samq_gemm_fp4, gemm)}


@pytest.mark.parametrize("name,change,code", [
    ("quant", {"x": None}, -1), ("quant", {"codes": None}, -1), ("quant", {"K": 0}, -1), ("quant", {"M": -1}, -1), ("quant", {"dtype": 9}, -1),
    ("quant", {"fmt": 2}, -1), ("quant", {"g": 3.0}, -1), ("quant", {"g": 0.0}, -1), ("quant", {"g": -2.0}, -1), ("quant", {"g": float("nan")}, -1),
    ("quant", {"g": 2.0 ** 65}, -1), ("quant", {"fmt": _lib.FP4_MX, "g": 2.0}, -1), ("quant", {"ldx": 63}, -1), ("quant", {"ldq": 31}, -1),
    ("quant", {"ldq": 1 << 20}, -1), ("quant", {"scales": (1 << 20) + 8}, -3), ("quant", {"x": (1 << 20) + 1}, -3),
    ("norm", {"x": None}, -1), ("norm", {"w": None}, -1), ("norm", {"K": 0}, -1), ("norm", {"K": 32769, "ldx": 32769}, -6), ("norm", {"eps": -1.0}, -1),
    ("norm", {"eps": float("nan")}, -1), ("norm", {"n_bits": 1}, -1), ("norm", {"n_bits": 9}, -1), ("norm", {"dtype": 3}, -1),
    ("norm", {"r": 1 << 20, "ldr": 64}, -1), ("norm", {"h": 1 << 20, "ldo": 64}, -1), ("norm", {"r": 1 << 20, "ldr": 64, "h": 1 << 20, "ldo": 63}, -1),
    ("norm", {"ldx": 60}, -1), ("norm", {"w": (1 << 20) + 1}, -3),
    ("gemm", {"A": None}, -1), ("gemm", {"sw": None}, -1), ("gemm", {"out": None}, -1), ("gemm", {"N": 0}, -1), ("gemm", {"K": -1}, -1),
    ("gemm", {"fmt": 5}, -1), ("gemm", {"act": 4}, -1), ("gemm", {"odt": _lib.I32}, -1), ("gemm", {"lda": 16}, -1), ("gemm", {"ldo": 7}, -1),
    ("gemm", {"res": 1 << 20, "ldr": 7}, -1), ("gemm", {"lda": 40}, -3), ("gemm", {"W": (1 << 20) + 8}, -3), ("gemm", {"sa": (1 << 20) + 4}, -3),
    ("linear", {"x": None}, -1), ("linear", {"M": 33}, -5), ("linear", {"M": 33, "ws": 1 << 20, "ws_bytes": 33 * 32 + 2047}, -5),
    ("linear", {"M": 33, "ws": (1 << 20) + 8, "ws_bytes": 1 << 20}, -5), ("linear", {"odt": _lib.F32}, -5), ("linear", {"odt": _lib.I32}, -1), ("linear", {"ldx": 63}, -1), ("linear", {"x": (1 << 20) + 1}, -3), ("linear", {"W": None}, -1),
    ("linear", {"sw": (1 << 20) + 8}, -3), ("linear", {"dtype": _lib.I32}, -1), ("linear", {"K": 0}, -1), ("linear", {"fmt": -1}, -1),
    ("gemm", {"out": (1 << 20) + 1}, -3), ("gemm", {"M": 1 << 31}, -6),
])
def test_entry_points_refuse_bad_arguments(name, change, code):
    built_library()
    lib = _lib.load()
    fn, args = _calls(lib)[name]
    assert fn(*dict(args, **change).values()) == code
    assert lib.samq_last_error_string() != b""


def test_no_rows_are_no_work():
    built_library()
    lib = _lib.load()
    for fn, args in _calls(lib).values():
        assert fn(*dict(args, M=0).values()) == 0


@pytest.mark.parametrize("name", ["gemm_fp4.cu", "gemm_fp4_pair.cu", "fp4_gemm.cuh"])
def test_loops_of_whole_warps_wait_as_a_warp(name):
    """A wait that ran out must send all lanes of a warp the same way: the loops of these kernels run warp-wide instructions
    behind their waits, so none polls a barrier lane by lane (the last join, with no such instruction behind it, is the
    cluster form)."""
    with open(os.path.join(os.path.dirname(_lib.__file__), "csrc", name)) as f:
        code = re.sub(r"//[^\n]*", "", f.read())
    assert "mbar_wait_warp(" in code and not re.search(r"\bmbar_(try_)?wait\(", code)


@pytest.mark.parametrize("change,code", [({"g": 3.0}, -1), ({"g": 0.0}, -1), ({"g": float("nan")}, -1), ({"g": 2.0 ** 65}, -1),
                                         ({"fmt": _lib.FP4_MX, "g": 2.0}, -1), ({"x": None}, -1), ({"M": 0}, 0), ({"M": 33}, -5)])
def test_layer_with_an_activation_scale_refuses_bad_arguments(change, code):
    built_library()
    lib = _lib.load()
    args = dict(_calls(lib)["linear"][1])
    args = dict(list(args.items())[:3] + [("g", 0.5)] + list(args.items())[3:])        # behind x, dtype and ldx
    assert lib.samq_linear_fp4_ex(*dict(args, **change).values()) == code


def test_layer_state_keeps_its_scales():
    layer = FP4Linear(32, 16, True, "nvfp4")
    assert layer.calibrate(1e-4, 5e3) == layer.act_global_scale == ops.fp4_global_scale(1e-4)
    other = FP4Linear(32, 16, True, "nvfp4")
    other.load_state_dict(layer.state_dict())
    assert (other.act_global_scale, other.output_global_scale) == (layer.act_global_scale, ops.fp4_global_scale(5e3))
    mx = FP4Linear(32, 16, True, "mxfp4")
    assert mx.calibrate(1e-4) == 1.0
    with pytest.raises(ValueError):
        layer.calibrate(float("inf"))


def test_kernels_of_a_layer():
    built_library()
    kernels = _lib.load().samq_linear_fp4_kernels
    need = _lib.load().samq_linear_fp4_workspace_bytes
    assert kernels(_lib.FP4_NV, _lib.BF16, _lib.BF16, 32, 640, 1280, 0) == 1
    assert kernels(_lib.FP4_NV, _lib.BF16, _lib.F32, 1, 640, 1280, 1 << 20) == 2 and kernels(_lib.FP4_MX, _lib.F16, _lib.F16, 33, 640, 1280, 1 << 20) == 2
    for ws, count in ((0, 1), (need(_lib.FP4_NV, 32, 20480) - 1, 1), (need(_lib.FP4_NV, 32, 20480), 2)):       # (a share of 10 blocks at least)
        assert kernels(_lib.FP4_NV, _lib.BF16, _lib.BF16, 32, 40000, 20480, ws) == count
    assert kernels(9, _lib.BF16, _lib.BF16, 1, 1, 1, 0) == 0 and kernels(_lib.FP4_NV, _lib.BF16, _lib.BF16, 0, 1, 1, 0) == 0


@pytest.mark.parametrize("name,change", [("gemm", {"alpha": float("inf")}), ("gemm", {"alpha": float("nan")}), ("linear", {"alpha": -float("inf")}),
                                         ("linear", {"alpha": 2.0 ** 128})])
def test_scales_whose_product_leaves_fp32_are_refused(name, change):
    """An infinite alpha would turn the sums that are zero into NaN."""
    built_library()
    lib = _lib.load()
    fn, args = _calls(lib)[name]
    assert fn(*dict(args, **change).values()) == -1 and b"alpha" in lib.samq_last_error_string()
    args = dict(_calls(lib)["linear"][1], alpha=2.0 ** 64)
    args = dict(list(args.items())[:3] + [("g", 2.0 ** 64)] + list(args.items())[3:])
    assert lib.samq_linear_fp4_ex(*args.values()) == -1 and b"alpha" in lib.samq_last_error_string()


@pytest.mark.parametrize("absmax,g", [(5e-324, 2.0 ** -64), (1e-320, 2.0 ** -64), (2688.0 * 2.0 ** -64, 2.0 ** -64), (2689.0 * 2.0 ** -64, 2.0 ** -63),
                                      (2688.0 * 2.0 ** 63, 2.0 ** 63), (1e308, 2.0 ** 64)])
def test_global_scale_at_its_ends(absmax, g):
    assert ops.fp4_global_scale(absmax) == g


def test_pickled_layers_without_activation_scales_have_ones():
    layer = FP4Linear(32, 16, True, "nvfp4")
    for name in ("act_global_scale", "output_global_scale"):
        del layer.__dict__[name]
    again = pickle.loads(pickle.dumps(layer))
    assert again.act_global_scale == again.output_global_scale == 1.0

"""Tensor-level wrappers over the C ABI (include/samq.h).

Each function takes CUDA tensors, allocates the outputs with torch (the library itself never
allocates), passes raw pointers plus the current CUDA stream through ctypes and returns the
outputs.  CPU tensors are rejected: this package has no CPU compute path.
"""
from __future__ import annotations

import ctypes
import math
import weakref
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import (ACT_GELU, ACT_NONE, BF16, F16, F32, GRAN_GROUP, GRAN_ROW, GRAN_TENSOR, HAD_FULL,
                   HAD_NONE, HAD_PARTIAL, I32, HadamardSpec, QuantPrologue)

_DTYPE_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}
_OUT_CODE = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32, torch.int32: I32}

# reference strings (RTN_quantization/per_tensor_channel_group.py:130-140,178-192) -> enum
ACT_GRANULARITY = {"per_token": GRAN_ROW, "per_tensor": GRAN_TENSOR, "per_group_token": GRAN_GROUP}
WEIGHT_GRANULARITY = {"per_channel": GRAN_ROW, "per_tensor": GRAN_TENSOR, "per_group": GRAN_GROUP}


@dataclass
class Hadamard:
    """Online transform applied before quantization (see ``samq_hadamard_spec``).

    mode: "full" (quarot/utils.py:257-261) or "partial" (:263-289)
    had_k / hadk: the explicit Hadamard factor of ``get_hadK`` (1 / None for powers of two)
    had_dim: head width for the partial transform
    signs: optional int8 [K] of +-1 multiplied in before the transform
    """

    mode: str
    had_k: int = 1
    hadk: Optional[torch.Tensor] = None
    had_dim: int = 0
    signs: Optional[torch.Tensor] = None


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: sam_quantization_b200 has no CPU compute path")


def _stream() -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t: Optional[torch.Tensor]) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


_status_words = {}

# ---- launch accounting and optional per-kernel timing (used by bench.py) -----------------------
_launches = 0
_timing_on = False
_timing_records = []          # (kind, start_event, end_event, work, detail)
_COUNTED_IN_OPS = ("gemm_i8", "gemm_fp4", "linear_fp4")      # kinds whose work is operations; the others' is bytes
_valid_rows = {}              # (data_ptr, numel) of a row map -> rows that are not padding


def reset_counters() -> None:
    global _launches
    _launches = 0


def launch_count() -> int:
    """CUDA kernels of this library launched since ``reset_counters()``."""
    return _launches


def enable_kernel_timing(on: bool) -> None:
    """Bracket every C-ABI launch with CUDA events on the launching stream."""
    global _timing_on
    _timing_on = bool(on)
    _timing_records.clear()


def kernel_timing_summary() -> dict:
    """{kind: {"ms", "launches", "ops" | "bytes"}} summed over the bracketed launches
    (synchronises).  ``ops`` = 2*M*N*K per GEMM (int8 or 4-bit, the 4-bit layer too), ``bytes`` = the algorithmic bytes of K1 (source rows
    actually read x element size + codes + scales).  The GEMM entry also carries ``bytes_alg`` (the
    algorithmic M*K + N*K + out_bytes*M*N) and ``"gemm_shapes"`` maps "KxN" to launches and total rows."""
    torch.cuda.synchronize()
    out = {}
    shapes = {}
    for kind, e0, e1, work, detail in _timing_records:
        d = out.setdefault(kind, {"ms": 0.0, "launches": 0, "ops": 0.0, "bytes": 0.0})
        ms = e0.elapsed_time(e1)
        d["ms"] += ms
        d["launches"] += 1
        d["ops" if kind in _COUNTED_IN_OPS else "bytes"] += work
        if kind == "gemm_i8" and detail is not None:
            M, N, K, out_bytes = detail
            d["bytes_alg"] = d.get("bytes_alg", 0.0) + M * K + N * K + out_bytes * M * N
            sh = shapes.setdefault(f"{K}x{N}", {"launches": 0, "rows": 0, "ms": 0.0, "ops": 0.0})
            sh["launches"] += 1
            sh["rows"] += M
            sh["ms"] += ms
            sh["ops"] += work
    if shapes:
        out["gemm_shapes"] = shapes
    return out


class _Timed:
    def __init__(self, kind, work, kernels=1, detail=None):
        self.kind, self.work, self.kernels, self.detail = kind, work, kernels, detail

    def __enter__(self):
        global _launches
        _launches += self.kernels
        if _timing_on:
            self.e0 = torch.cuda.Event(enable_timing=True)
            self.e1 = torch.cuda.Event(enable_timing=True)
            self.e0.record()
        return self

    def __exit__(self, *exc):
        if _timing_on:
            self.e1.record()
            _timing_records.append((self.kind, self.e0, self.e1, self.work, self.detail))
        return False


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 that GEMM kernels raise when one of their bounded waits ran out."""
    key = torch.device(device).index if torch.device(device).index is not None else torch.cuda.current_device()
    if key not in _status_words:
        _status_words[key] = torch.zeros(1, dtype=torch.int32, device=f"cuda:{key}")
    return _status_words[key]


def check_status(device=None) -> None:
    """Synchronise and raise if any GEMM kernel on ``device`` reported a timed-out wait."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = status_word(dev)
    if int(word.item()) != 0:
        word.zero_()
        raise RuntimeError("samq GEMM kernel gave up on a bounded wait (pipeline stalled)")


def _as_rows(x: torch.Tensor) -> Tuple[torch.Tensor, int, int, int]:
    """View x as [M, K] with a row stride; copies only if the last dim is not contiguous."""
    K = x.shape[-1]
    if K and x.is_contiguous():
        return x, x.numel() // K, K, K
    if x.dim() == 2 and x.stride(1) == 1 and x.stride(0) >= K:
        return x, x.shape[0], K, x.stride(0)
    x2 = x.reshape(-1, K)
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) != K):
        x2 = x2.contiguous()
    return x2, x2.shape[0], K, K


def _spec(had: Optional[Hadamard], keep: list) -> Optional[HadamardSpec]:
    if had is None:
        return None
    mode = {"full": HAD_FULL, "partial": HAD_PARTIAL, "none": HAD_NONE}[had.mode]
    hadk = None
    if had.had_k > 1:
        if had.hadk is None:
            raise ValueError("had_k > 1 needs the hadk matrix")
        hadk = had.hadk.to(dtype=torch.float32).contiguous()
        _require_cuda(hadk, "hadk")
        keep.append(hadk)
    signs = None
    if had.signs is not None:
        signs = had.signs.to(dtype=torch.int8).contiguous()
        _require_cuda(signs, "signs")
        keep.append(signs)
    return HadamardSpec(mode, int(had.had_k), 0 if hadk is None else hadk.data_ptr(), int(had.had_dim),
                        0 if signs is None else signs.data_ptr())


def hadamard_layer_norm_fused(x: torch.Tensor, hadamard: "Hadamard", as_dtype: Optional[torch.dtype] = None) -> bool:
    """True when ``quantize(x, GRAN_ROW, hadamard=..., layer_norm=...)`` runs as one kernel: a full
    power-of-two transform over fp16 rows of 1024 elements (codes and scales only)."""
    return (hadamard is not None and hadamard.mode == "full" and int(hadamard.had_k) == 1 and x.dtype == torch.float16 and
            (as_dtype is None or as_dtype == torch.float16) and x.shape[-1] == 1024)


def quantize(x: torch.Tensor, granularity: int = GRAN_ROW, group_size: Optional[int] = None,
             divisor: Optional[torch.Tensor] = None, hadamard: Optional[Hadamard] = None,
             codes: bool = True, fake_quant: bool = False, transformed: bool = False, n_bits: int = 8,
             row_map: Optional[torch.Tensor] = None, layer_norm=None, as_dtype: Optional[torch.dtype] = None):
    """Run K1 on ``x`` ([..., K]; fp16 / bf16 / fp32).

    Returns a dict with the requested outputs: ``q`` int8 [..., K], ``scale`` fp32
    ([...] | [1] | [..., K/group]), ``fq`` (fake-quantized) and ``tx`` (input after the
    prologue / divisor / Hadamard), both in the tensor dtype.

    Prologue fused into the same kernel (see ``samq_quant_prologue``): ``row_map`` int32 [M_out]
    gathers source rows (negative = a zero row) and makes the outputs ``[M_out, ...]``;
    ``layer_norm=(weight, bias, eps)`` normalises each source row first; ``as_dtype=torch.float16``
    reads a bf16 ``x`` as the fp16 tensor the model would cast it to.
    """
    _require_cuda(x, "x")
    if x.dtype not in _DTYPE_CODE:
        raise TypeError(f"unsupported dtype {x.dtype}")
    lib = _lib.load()
    lead = x.shape[:-1]
    x2, M, K, ldx = _as_rows(x)
    tdtype = x.dtype
    pro = None
    keep_pro = []
    if row_map is not None or layer_norm is not None or (as_dtype is not None and as_dtype != x.dtype):
        pro = QuantPrologue(0, 0, 0, 0.0, -1)
        if row_map is not None:
            _require_cuda(row_map, "row_map")
            if row_map.dtype != torch.int32 or not row_map.is_contiguous():
                raise TypeError("row_map must be a contiguous int32 tensor")
            pro.row_map = row_map.data_ptr()
            M = row_map.numel()
            lead = (M,)
        if as_dtype is not None and as_dtype != x.dtype:
            if not (x.dtype == torch.bfloat16 and as_dtype == torch.float16):
                raise TypeError("as_dtype only reads bf16 storage as an fp16 tensor")
            pro.src_dtype = _DTYPE_CODE[x.dtype]
            tdtype = as_dtype
        if layer_norm is not None:
            ln_w, ln_b, ln_eps = layer_norm
            ln_w = ln_w.detach().to(device=x.device, dtype=tdtype).contiguous()
            ln_b = ln_b.detach().to(device=x.device, dtype=tdtype).contiguous()
            keep_pro += [ln_w, ln_b]
            pro.ln_weight, pro.ln_bias, pro.ln_eps = ln_w.data_ptr(), ln_b.data_ptr(), float(ln_eps)
    g = int(group_size) if granularity == GRAN_GROUP else 0
    if granularity == GRAN_GROUP:
        if not isinstance(group_size, int):
            raise AssertionError("group_size must be an integer")
        if K % g != 0:
            raise AssertionError(f"Last dimension ({K}) must be divisible by group_size ({g})")
    out = {}
    dev = x.device
    q = torch.empty((M, K), dtype=torch.int8, device=dev) if codes else None
    if granularity == GRAN_ROW:
        scale = torch.empty((M,), dtype=torch.float32, device=dev)
    elif granularity == GRAN_TENSOR:
        scale = torch.empty((1,), dtype=torch.float32, device=dev)
    else:
        scale = torch.empty((M, K // g), dtype=torch.float32, device=dev)
    fq = torch.empty((M, K), dtype=tdtype, device=dev) if fake_quant else None
    tx = torch.empty((M, K), dtype=tdtype, device=dev) if transformed else None
    ws_bytes = int(lib.samq_quant_workspace_bytes(granularity))
    ws = torch.empty((max(ws_bytes, 4) // 4,), dtype=torch.int32, device=dev) if ws_bytes else None
    keep = []
    if divisor is not None:
        divisor = divisor.to(device=dev, dtype=tdtype).contiguous()
        if divisor.numel() != K:
            raise ValueError("divisor must have K elements")
    spec = _spec(hadamard, keep)
    rows_read = M
    if _timing_on and row_map is not None:                # padding rows (negative map entries) read nothing
        key = (row_map.data_ptr(), row_map.numel())
        if key not in _valid_rows:
            _valid_rows[key] = int((row_map >= 0).sum().item())
        rows_read = _valid_rows[key]
    nbytes = rows_read * K * x.element_size() + M * ((K if codes else 0) + (K * x.element_size() if fake_quant else 0)
                                                     + (K * x.element_size() if transformed else 0)) + scale.numel() * 4
    with torch.cuda.device(dev), _Timed("act_quant", nbytes, 3 if granularity == GRAN_TENSOR else 1):
        _lib.check(lib.samq_act_quant_i8_ex(
            _ptr(x2), _DTYPE_CODE[tdtype], M, K, ldx,
            ctypes.byref(pro) if pro is not None else None, _ptr(divisor),
            ctypes.byref(spec) if spec is not None else None,
            granularity, g, int(n_bits), _ptr(q), _ptr(scale), _ptr(fq), _ptr(tx),
            _ptr(ws), ws_bytes, _stream()))
    if codes:
        out["q"] = q.view(*lead, K)
    if granularity == GRAN_ROW:
        out["scale"] = scale.view(*lead)
    elif granularity == GRAN_TENSOR:
        out["scale"] = scale
    else:
        out["scale"] = scale.view(*lead, K // g)
    if fake_quant:
        out["fq"] = fq.view(*lead, K)
    if transformed:
        out["tx"] = tx.view(*lead, K)
    return out


def quantize_weight(w: torch.Tensor, granularity: int = GRAN_ROW, group_size: Optional[int] = None,
                    codes: bool = True, fake_quant: bool = False, n_bits: int = 8):
    """Run K3 (weight quantization) on ``w`` [N, K] through ``samq_weight_quant_i8``."""
    _require_cuda(w, "w")
    if w.dim() != 2:
        raise AssertionError("weight must be 2-D")
    if w.dtype not in _DTYPE_CODE:
        raise TypeError(f"unsupported dtype {w.dtype}")
    lib = _lib.load()
    w2, N, K, ldw = _as_rows(w)
    g = int(group_size) if granularity == GRAN_GROUP else 0
    if granularity == GRAN_GROUP:
        if not isinstance(group_size, int):
            raise AssertionError("group_size must be an integer")
        if K % g != 0:
            raise AssertionError(f"in_features ({K}) must be divisible by group_size ({g})")
    dev = w.device
    q = torch.empty((N, K), dtype=torch.int8, device=dev) if codes else None
    shape = {GRAN_ROW: (N,), GRAN_TENSOR: (1,), GRAN_GROUP: (N, K // g if g else 1)}[granularity]
    scale = torch.empty(shape, dtype=torch.float32, device=dev)
    fq = torch.empty((N, K), dtype=w.dtype, device=dev) if fake_quant else None
    ws_bytes = int(lib.samq_quant_workspace_bytes(granularity))
    ws = torch.empty((max(ws_bytes, 4) // 4,), dtype=torch.int32, device=dev) if ws_bytes else None
    with torch.cuda.device(dev), _Timed("weight_quant", N * K * (w.element_size() + 1), 3 if granularity == GRAN_TENSOR else 1):
        _lib.check(lib.samq_weight_quant_i8(
            _ptr(w2), _DTYPE_CODE[w.dtype], N, K, ldw, granularity, g, int(n_bits),
            _ptr(q), _ptr(scale), _ptr(fq), _ptr(ws), ws_bytes, _stream()))
    out = {"scale": scale}
    if codes:
        out["q"] = q
    if fake_quant:
        out["fq"] = fq
    return out


GEMM_GROUP_MULTIPLE = 32        # one tcgen05.mma covers 32 columns of K
GEMM_MAX_GROUPS = 160


def check_gemm_group_size(in_features: int, group_size) -> None:
    """Raise early (at module construction) for a group size the grouped int8 GEMM cannot run: the
    reference's float path accepts any divisor of the width; the tensor-core path needs groups of a
    multiple of 32 columns and at most 160 groups per row."""
    assert type(group_size) == int, "group_size must be an integer"
    assert in_features % group_size == 0, f"in_features ({in_features}) must be divisible by group_size ({group_size})"
    if group_size % GEMM_GROUP_MULTIPLE != 0 or in_features // group_size > GEMM_MAX_GROUPS:
        raise ValueError(f"group_size={group_size} with in_features={in_features}: the int8 GEMM needs group sizes that are "
                         f"multiples of {GEMM_GROUP_MULTIPLE} and at most {GEMM_MAX_GROUPS} groups per row")


GEMM_PAIR_NEVER, GEMM_PAIR_AUTO, GEMM_PAIR_ALWAYS = 0, 1, 2


def set_gemm_pair_mode(mode: int) -> int:
    """Choose the K2 implementation: single CTAs, CTA pairs (tcgen05 cta_group::2), or by size.

    Returns the previous mode.  Both implementations give bit-identical results.
    """
    prev = _lib.load().samq_gemm_set_pair_mode(int(mode))
    if prev < 0:
        raise ValueError(f"unknown GEMM pair mode {mode}")
    return prev


_bias_cache = {}


def _bias_as(bias: torch.Tensor, dtype: torch.dtype, dev) -> torch.Tensor:
    """``bias`` flattened in the epilogue's parameter dtype.  A layer whose output dtype differs from its
    bias dtype (qkv storing bf16 for the attention) would otherwise launch a conversion kernel on every
    call; the converted copy is cached until the bias changes (new storage or an in-place update)."""
    if bias.dtype == dtype and bias.device == dev and bias.dim() == 1 and bias.is_contiguous():
        return bias
    key = (id(bias), bias.data_ptr(), bias._version, dtype, str(dev))
    hit = _bias_cache.get(key)
    if hit is None or hit[0]() is not bias:              # the weak reference guards against a recycled id / address
        if len(_bias_cache) > 4096:
            _bias_cache.clear()
        hit = (weakref.ref(bias), bias.detach().reshape(-1).to(device=dev, dtype=dtype).contiguous())
        _bias_cache[key] = hit
    return hit[1]


def gemm_i8(a_q: torch.Tensor, w_q: torch.Tensor,
            a_scale: Optional[torch.Tensor] = None, w_scale: Optional[torch.Tensor] = None,
            a_gran: int = GRAN_ROW, w_gran: int = GRAN_ROW, group_size: int = 0,
            bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
            activation: int = ACT_NONE, out_dtype: torch.dtype = torch.float16,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Run K2: ``act(dequant(a_q @ w_q.T) + bias) + residual`` -> [..., N] of ``out_dtype``.

    ``out_dtype=torch.int32`` returns the raw accumulators (no scales / bias allowed).
    """
    _require_cuda(a_q, "a_q")
    _require_cuda(w_q, "w_q")
    if a_q.dtype != torch.int8 or w_q.dtype != torch.int8:
        raise TypeError("a_q and w_q must be int8")
    lib = _lib.load()
    lead = a_q.shape[:-1]
    a2, M, K, lda = _as_rows(a_q)
    if w_q.dim() != 2 or w_q.shape[1] != K:
        raise ValueError(f"w_q must be [N, {K}]")
    w2, N, _, ldw = _as_rows(w_q)
    dev = a_q.device
    if out is None:
        out = torch.empty((M, N), dtype=out_dtype, device=dev)
    else:
        if out.dtype != out_dtype or out.shape[-1] != N or out.numel() != M * N or not out.is_contiguous():
            raise ValueError("out has the wrong dtype, shape or layout")
    param_dtype = torch.float32 if out_dtype in (torch.float32, torch.int32) else out_dtype
    if bias is not None:
        bias = _bias_as(bias, param_dtype, dev)
        if bias.numel() != N:
            raise ValueError("bias must have N elements")
    ldr = 0
    if residual is not None:
        _require_cuda(residual, "residual")
        if residual.dtype != out_dtype:
            raise TypeError("residual must have the output dtype")
        residual, rm, rn, ldr = _as_rows(residual)
        if rm != M or rn != N:
            raise ValueError("residual must be [..., N] with the rows of a_q")
    if a_scale is not None:
        a_scale = a_scale.to(device=dev, dtype=torch.float32).contiguous()
    if w_scale is not None:
        w_scale = w_scale.to(device=dev, dtype=torch.float32).contiguous()
    with torch.cuda.device(dev), _Timed("gemm_i8", 2.0 * M * N * K, detail=(M, N, K, out.element_size())):
        _lib.check(lib.samq_gemm_i8(
            _ptr(a2), lda, _ptr(w2), ldw, M, N, K,
            _ptr(a_scale), a_gran, _ptr(w_scale), w_gran, int(group_size or 0),
            _ptr(bias), _ptr(residual), ldr, activation,
            _ptr(out), _OUT_CODE[out_dtype], N, _ptr(status_word(dev)), _stream()))
    return out.view(*lead, N)


# ---- RMS norm with an 8-bit output -----------------------------------------------------------------
#
# The calls below serve single tokens too, where the host's time per call is the call's time: pointers go to ctypes
# as plain integers, and the device is only switched when it is not the current one.

def _data_ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


def _call(dev: torch.device, kind: str, work: float, fn, *args, kernels: int = 1) -> None:
    """``fn(*args, stream)`` on the current stream of ``dev``, counted (and timed) like every launch."""
    if _timing_on or torch.cuda.current_device() != dev.index:
        with torch.cuda.device(dev), _Timed(kind, work, kernels):
            _lib.check(fn(*args, torch.cuda.current_stream().cuda_stream))
        return
    global _launches
    _launches += kernels
    code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if code:
        _lib.check(code)


def _status_ptr(dev: torch.device) -> int:
    word = _status_words.get(dev.index)
    return (status_word(dev) if word is None else word).data_ptr()


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                      codes: bool = True, fake_quant: bool = False, n_bits: int = 8,
                      residual_out: Optional[torch.Tensor] = None) -> dict:
    """RMS norm of ``x`` ([..., K]; fp16 / bf16 / fp32), or of ``x + residual``, quantized per row in the same pass
    (``samq_rms_norm_quant_i8``).

    Returns a dict with ``q`` int8 [..., K] (unless ``codes=False``) and ``scale`` fp32 [...], what ``gemm_i8`` takes,
    ``fq`` (with ``fake_quant``) the values ``q * scale`` in the tensor dtype and, with a ``residual``, ``residual``:
    the sum ``x + residual`` in the tensor dtype, in a new tensor or in ``residual_out`` (which may be ``residual`` or
    ``x`` itself).  The normed value is quantized from fp32, without a rounding to the tensor dtype in between.  A ``weight``
    of another dtype is converted to that of ``x`` (an fp32 weight is rounded to it), by a kernel in every call."""
    if not x.is_cuda:
        _require_cuda(x, "x")
    dtype, dev, shape = x.dtype, x.device, x.shape
    code = _DTYPE_CODE.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}")
    x2, M, K, ldx = _as_rows(x)
    if weight.numel() != K:
        raise ValueError("weight must have K elements")
    if weight.dtype != dtype or weight.device != dev or not weight.is_contiguous():
        weight = weight.detach().reshape(-1).to(device=dev, dtype=dtype).contiguous()
    res2 = h2 = h = None
    ldr = ldo = 0
    if residual is not None:
        if residual.shape != shape or residual.dtype != dtype or residual.device != dev:
            raise ValueError("residual must have the shape, dtype and device of x")
        res2, _, _, ldr = _as_rows(residual)
        if residual_out is None:
            h = h2 = torch.empty_like(x, memory_format=torch.contiguous_format)
            ldo = K
        else:
            h = residual_out
            h2, hm, hk, ldo = _as_rows(h)
            if h.dtype != dtype or h.device != dev or hm != M or hk != K or h2.data_ptr() != h.data_ptr():
                raise ValueError("residual_out must be rows of K contiguous elements with the shape, dtype and device of x")
    elif residual_out is not None:
        raise ValueError("residual_out without a residual")
    out = {"scale": x.new_empty(shape[:-1], dtype=torch.float32)}
    q = fq = None
    if codes:
        out["q"] = q = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    if fake_quant:
        out["fq"] = fq = torch.empty_like(x, memory_format=torch.contiguous_format)
    if h is not None:
        out["residual"] = h
    nbytes = 0 if not _timing_on else \
        M * K * (dtype.itemsize * (1 + (2 if h is not None else 0) + (1 if fake_quant else 0)) + (1 if codes else 0)) + 4 * M
    _call(dev, "rms_norm_quant", nbytes, _lib.load().samq_rms_norm_quant_i8, x2.data_ptr(), _data_ptr(res2), weight.data_ptr(), code, M, K,
          ldx, ldr, eps, n_bits, _data_ptr(h2), ldo, _data_ptr(q), out["scale"].data_ptr(), _data_ptr(fq))
    return out


# ---- microscaled 4-bit floating point ----------------------------------------------------------------

FP4_FORMATS = {"mxfp4": _lib.FP4_MX, "nvfp4": _lib.FP4_NV}
FP4_BLOCK = {"mxfp4": 32, "nvfp4": 16}
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def fp4_scale_shape(fmt: str, rows: int, K: int) -> Tuple[int, ...]:
    """Shape of the scale tiles of a [rows, K] operand (include/samq.h gives their order)."""
    return ((rows + 127) // 128, (K + 255) // 256 * (64 // FP4_BLOCK[fmt]), 32, 4, 4)


def fp4_global_scale(absmax: float) -> float:
    """The power of two that brings the largest nvfp4 block scale of a tensor with this largest magnitude into
    (224, 448], the top of e4m3; 1.0 for a tensor of zeros."""
    absmax = float(absmax)
    if not math.isfinite(absmax):
        raise ValueError("a global scale needs a finite largest magnitude")
    if absmax <= 0.0:
        return 1.0
    if absmax <= 6.0 * 448.0 * 2.0 ** -64:
        return 2.0 ** -64
    return min(2.0 ** math.ceil(math.log2(absmax / (6.0 * 448.0))), 2.0 ** 64)


class Fp4Tensor:
    """A [rows, K] operand in microscaled 4-bit floating point: ``codes`` uint8 [rows, pitch], ``scales`` uint8 in the
    tiles of ``fp4_scale_shape``, ``fmt`` "mxfp4" or "nvfp4", ``global_scale`` a float that multiplies every value."""

    __slots__ = ("codes", "scales", "rows", "K", "fmt", "global_scale")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, K: int, fmt: str, global_scale: float = 1.0):
        if fmt not in FP4_FORMATS:
            raise ValueError(f"Invalid 4-bit format: {fmt}")
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if codes.dim() != 2 or codes.shape[0] != rows or codes.shape[1] < (K + 1) // 2 or codes.stride(1) != 1:
            raise ValueError(f"codes must be [{rows}, >= {(K + 1) // 2}] with contiguous rows")
        if scales.device != codes.device or not scales.is_contiguous() or scales.shape != fp4_scale_shape(fmt, rows, K):
            raise ValueError(f"scales must be a contiguous {fp4_scale_shape(fmt, rows, K)} tensor on the device of codes")
        self.codes, self.scales, self.rows, self.K, self.fmt, self.global_scale = codes, scales, rows, K, fmt, float(global_scale)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype = torch.float32) -> torch.Tensor:
        """The values [rows, K], the global scale included, rounded once to ``dtype`` if that scale is a power of two (off the
        hot path: plain torch)."""
        b = FP4_BLOCK[self.fmt]
        table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1), device=self.device)
        v = table[torch.stack((self.codes & 15, self.codes >> 4), -1).flatten(1)[:, :self.K].long()]
        nb = (self.K + b - 1) // b
        byte = self.scales.permute(0, 3, 2, 1, 4).reshape(-1, 4 * self.scales.shape[1])[:self.rows, :nb]
        s = byte.contiguous().view(torch.float8_e8m0fnu if self.fmt == "mxfp4" else torch.float8_e4m3fn).float()
        return (v * s.repeat_interleave(b, 1)[:, :self.K] * self.global_scale).to(dtype)


def quantize_fp4(x: torch.Tensor, fmt: str = "nvfp4", global_scale: float = 1.0, fake_quant: bool = False) -> dict:
    """Quantize ``x`` ([..., K]; fp16 / bf16 / fp32) to microscaled 4-bit floating point (``samq_quant_fp4``).

    Returns a dict with ``q``, an ``Fp4Tensor`` of the rows of ``x``, and with ``fake_quant`` ``fq``, the values it
    stands for in the dtype and shape of ``x``.  ``global_scale`` (nvfp4) is a power of two, see ``fp4_global_scale``."""
    if not x.is_cuda:
        _require_cuda(x, "x")
    dev = x.device
    code = _DTYPE_CODE.get(x.dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {x.dtype}")
    fcode = FP4_FORMATS.get(fmt)
    if fcode is None:
        raise ValueError(f"Invalid 4-bit format: {fmt}")
    x2, M, K, ldx = _as_rows(x)
    pitch = (K + 31) // 32 * 16
    codes = x.new_empty((M, pitch), dtype=torch.uint8)
    scales = x.new_empty(fp4_scale_shape(fmt, M, K), dtype=torch.uint8)
    fq = torch.empty_like(x, memory_format=torch.contiguous_format) if fake_quant else None
    nbytes = 0 if not _timing_on else M * K * x.dtype.itemsize * (2 if fake_quant else 1) + codes.numel() + scales.numel()
    _call(dev, "quant_fp4", nbytes, _lib.load().samq_quant_fp4, x2.data_ptr(), code, M, K, ldx, fcode, global_scale, codes.data_ptr(), pitch,
          scales.data_ptr(), _data_ptr(fq))
    out = {"q": Fp4Tensor(codes, scales, M, K, fmt, global_scale)}
    if fake_quant:
        out["fq"] = fq
    return out


def _linear_args(N: int, M: int, bias, residual, out_dtype, dev):
    """Checked dtype code, bias and residual rows of a linear layer's epilogue, as ``gemm_i8`` takes them."""
    code = _DTYPE_CODE.get(out_dtype)
    if code is None:
        raise TypeError(f"unsupported out_dtype {out_dtype}")
    if bias is not None:
        if bias.dtype != out_dtype or bias.device != dev or not bias.is_contiguous():
            bias = bias.detach().to(device=dev, dtype=out_dtype).contiguous()
        if bias.numel() != N:
            raise ValueError("bias must have N elements")
    ldr = 0
    if residual is not None:
        if residual.device != dev:
            raise ValueError("residual must be on the device of the operands")
        if residual.dtype != out_dtype:
            raise TypeError("residual must have the output dtype")
        residual, rm, rn, ldr = _as_rows(residual)
        if rm != M or rn != N:
            raise ValueError("residual must be [..., N] with the rows of the activation")
    return code, bias, residual, ldr


def gemm_fp4(a: Fp4Tensor, w: Fp4Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
             activation: int = ACT_NONE, out_dtype: torch.dtype = torch.float16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(a @ w.T + bias) + residual`` -> [a.rows, w.rows] of ``out_dtype`` from two 4-bit operands of one format, on
    the tensor cores' block-scaled kinds (``samq_gemm_fp4``).  A ``bias`` of another dtype is converted to ``out_dtype``, by a
    kernel in every call."""
    ac, wc = a.codes, w.codes
    dev = ac.device
    if not ac.is_cuda:
        _require_cuda(ac, "a")
    if a.fmt != w.fmt or a.K != w.K or dev != wc.device:
        raise ValueError(f"operands must share format, K and device: {a.fmt} [{a.rows}, {a.K}] and {w.fmt} [{w.rows}, {w.K}]")
    M, N, K = a.rows, w.rows, a.K
    code, bias, residual, ldr = _linear_args(N, M, bias, residual, out_dtype, dev)
    if out is None:
        out = ac.new_empty((M, N), dtype=out_dtype)
    elif out.dtype != out_dtype or out.device != dev or out.shape[-1] != N or out.numel() != M * N or not out.is_contiguous():
        raise ValueError("out has the wrong dtype, device, shape or layout")
    _call(dev, "gemm_fp4", 2.0 * M * N * K, _lib.load().samq_gemm_fp4, ac.data_ptr(), ac.stride(0), a.scales.data_ptr(), wc.data_ptr(),
          wc.stride(0), w.scales.data_ptr(), M, N, K, FP4_FORMATS[a.fmt], a.global_scale * w.global_scale, _data_ptr(bias),
          _data_ptr(residual), ldr, activation, out.data_ptr(), code, N, _status_ptr(dev))
    return out


def linear_fp4(x: torch.Tensor, w: Fp4Tensor, bias: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
               activation: int = ACT_NONE, out_dtype: Optional[torch.dtype] = None, x_global_scale: float = 1.0) -> torch.Tensor:
    """``x`` ([..., K]) quantized to the format of ``w`` and multiplied with it:
    ``act(q(x) @ w.T + bias) + residual`` -> [..., N], of ``x.dtype`` unless ``out_dtype`` says otherwise.

    ``x_global_scale`` (nvfp4) is the power of two under which ``x`` is quantized: magnitudes beyond 2688 times it saturate,
    blocks below about 2^-6 times it lose resolution.  The default serves activations around 1; ``fp4_global_scale`` gives
    the scale for a calibrated largest magnitude.  ``bias`` as in ``gemm_fp4``."""
    if x.shape[-1] != w.K:
        raise ValueError(f"x must be [..., {w.K}]")
    if not x.is_cuda:
        _require_cuda(x, "x")
    N, K, dev, dtype, wc = w.rows, w.K, x.device, x.dtype, w.codes
    xcode, fcode = _DTYPE_CODE.get(dtype), FP4_FORMATS[w.fmt]
    if xcode is None:
        raise TypeError(f"unsupported dtype {dtype}")
    if dev != wc.device:
        raise ValueError("x must be on the device of w")
    lib = _lib.load()
    x2, M, _, ldx = _as_rows(x)
    if out_dtype is None:
        out_dtype = dtype
    code, bias, residual, ldr = _linear_args(N, M, bias, residual, out_dtype, dev)
    out = x.new_empty((*x.shape[:-1], N), dtype=out_dtype)
    ws, ws_bytes, kernels = None, 0, 1
    two = M > _lib.LINEAR_FP4_ONE_KERNEL_ROWS or code != xcode
    if two or (M + 8) * ((K + 255) // 256) > _lib.LINEAR_FP4_ONE_KERNEL_WORK:      # (the latter may use it)
        ws_bytes = lib.samq_linear_fp4_workspace_bytes(fcode, M, K)
        ws = x.new_empty((ws_bytes,), dtype=torch.uint8)
        kernels = 2 if two else lib.samq_linear_fp4_kernels(fcode, xcode, code, M, N, K, ws_bytes)
    _call(dev, "linear_fp4", 2.0 * M * N * K, lib.samq_linear_fp4_ex, x2.data_ptr(), xcode, ldx, x_global_scale, wc.data_ptr(), wc.stride(0), w.scales.data_ptr(),
          M, N, K, fcode, w.global_scale, _data_ptr(bias), _data_ptr(residual), ldr, activation, out.data_ptr(), code, N,
          _data_ptr(ws), ws_bytes, _status_ptr(dev), kernels=kernels)
    return out


def gemm_stall_selftest(a_q: torch.Tensor, w_q: torch.Tensor, skip_kblock: int = 0, wait_limit_cycles: int = 2_000_000) -> torch.Tensor:
    """Run ``samq_gemm_i8_stall_selftest``: the raw-int32 GEMM with one operand stage that the
    producer never fills, so that a bounded wait inside the kernel runs out.  The kernel returns on
    its own and raises the device status word (``check_status`` then raises); the returned tensor
    is incomplete."""
    _require_cuda(a_q, "a_q")
    lib = _lib.load()
    M, K = a_q.shape
    N = w_q.shape[0]
    out = torch.zeros((M, N), dtype=torch.int32, device=a_q.device)
    with torch.cuda.device(a_q.device):
        _lib.check(lib.samq_gemm_i8_stall_selftest(_ptr(a_q), a_q.stride(0), _ptr(w_q), w_q.stride(0), M, N, K, _ptr(out), N,
                                                   int(skip_kblock), int(wait_limit_cycles), _ptr(status_word(a_q.device)), _stream()))
    return out


def rel_pos_table(rel_pos_h: torch.Tensor, rel_pos_w: torch.Tensor, dtype, device) -> torch.Tensor:
    """The rows of ``rel_pos_h`` followed by those of ``rel_pos_w`` as one [J, d] matrix of
    ``dtype`` (J rounded up to a multiple of 8, zero rows at the end)."""
    rows = rel_pos_h.shape[0] + rel_pos_w.shape[0]
    J = (rows + 7) // 8 * 8
    tab = torch.zeros((J, rel_pos_h.shape[1]), dtype=dtype, device=device)
    tab[:rel_pos_h.shape[0]] = rel_pos_h.detach().to(device=device, dtype=dtype)
    tab[rel_pos_h.shape[0]:rows] = rel_pos_w.detach().to(device=device, dtype=dtype)
    return tab


def rel_pos_products(qkv: torch.Tensor, num_heads: int, table: torch.Tensor) -> torch.Tensor:
    """rel_all[head, token, j] = q[token, head, :] . table[j, :]: one batched tensor-core GEMM on
    strided views of ``qkv`` [tokens, 3C], no copy of q."""
    tokens, three_c = qkv.shape
    d = three_c // 3 // num_heads
    q_heads = qkv.view(tokens, 3, num_heads, d)[:, 0].permute(1, 0, 2)          # [heads, tokens, d], strides (d, 3C, 1)
    return torch.matmul(q_heads, table.t())                                      # [heads, tokens, J]


def attn_window_prep(qkv: torch.Tensor, H: int, W: int, num_heads: int, rel_pos_h: torch.Tensor,
                     rel_pos_w: torch.Tensor, scale: float, width: int, table: Optional[torch.Tensor] = None):
    """Augmented attention inputs for windows (``samq_attn_window_prep``): from ``qkv``
    [tokens, 3C] returns ``(q_aug, k_aug)``, each [tokens, heads, width].  ``table`` is an
    optional cached ``rel_pos_table`` of the two tables."""
    _require_cuda(qkv, "qkv")
    lib = _lib.load()
    tokens, three_c = qkv.shape
    d = three_c // 3 // num_heads
    if not qkv.is_contiguous():
        raise ValueError("qkv must be contiguous")
    if rel_pos_h.shape != (2 * H - 1, d) or rel_pos_w.shape != (2 * W - 1, d):
        raise ValueError("relative position tables must be [2H-1, d] and [2W-1, d]")
    if table is None:
        table = rel_pos_table(rel_pos_h, rel_pos_w, qkv.dtype, qkv.device)
    rel_all = rel_pos_products(qkv, num_heads, table)
    if not rel_all.is_contiguous():
        rel_all = rel_all.contiguous()
    qa = torch.empty((tokens, num_heads, width), dtype=qkv.dtype, device=qkv.device)
    ka = torch.empty((tokens, num_heads, width), dtype=qkv.dtype, device=qkv.device)
    with torch.cuda.device(qkv.device), _Timed("attn_prep", tokens * num_heads * (2 * d + 2 * width) * qkv.element_size()):
        _lib.check(lib.samq_attn_window_prep(_ptr(qkv), _ptr(rel_all), _DTYPE_CODE[qkv.dtype], tokens, rel_all.shape[-1],
                                             H, W, num_heads, d, float(scale), width, _ptr(qa), _ptr(ka), _stream()))
    return qa, ka


def attn_rel_bias(qkv: torch.Tensor, images: int, H: int, W: int, num_heads: int, rel_pos_h: torch.Tensor,
                  rel_pos_w: torch.Tensor, table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Explicit relative-position bias [images, heads, H*W, H*W] for global attention
    (``samq_attn_rel_bias``) from ``qkv`` [images*H*W, 3C]."""
    _require_cuda(qkv, "qkv")
    lib = _lib.load()
    tokens, three_c = qkv.shape
    L = H * W
    if tokens != images * L or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous [images*H*W, 3C] tensor")
    if table is None:
        table = rel_pos_table(rel_pos_h, rel_pos_w, qkv.dtype, qkv.device)
    rel_all = rel_pos_products(qkv, num_heads, table)
    if not rel_all.is_contiguous():
        rel_all = rel_all.contiguous()
    bias = torch.empty((images, num_heads, L, L), dtype=qkv.dtype, device=qkv.device)
    with torch.cuda.device(qkv.device), _Timed("attn_bias", bias.numel() * bias.element_size()):
        _lib.check(lib.samq_attn_rel_bias(_ptr(rel_all), _DTYPE_CODE[qkv.dtype], images, rel_all.shape[-1], H, W, num_heads,
                                          _ptr(bias), _stream()))
    return bias


def attn_global_supported(H: int, W: int, head_dim: int, dtype) -> bool:
    """Shapes ``samq_attn_global`` is built for: images of H x 64 tokens or windows up to 16 x 16."""
    shape_ok = (W == 64 and (H * W) % 128 == 0) or (W <= 16 and H <= 16)
    return shape_ok and head_dim in (64, 80) and dtype in (torch.float16, torch.bfloat16)


def attn_global(qkv: torch.Tensor, units: int, H: int, W: int, num_heads: int, rel_pos_h: torch.Tensor,
                rel_pos_w: torch.Tensor, scale: float, table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention with the decomposed relative-position bias on the tensor cores (``samq_attn_global``):
    ``qkv`` [units*H*W, 3C] -> [units*H*W, C], heads side by side; a unit is an image (W = 64) or a
    window (H, W <= 16).  Scores and bias stay on chip."""
    _require_cuda(qkv, "qkv")
    lib = _lib.load()
    tokens, three_c = qkv.shape
    C = three_c // 3
    d = C // num_heads
    L = H * W
    if tokens != units * L or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous [units*H*W, 3C] tensor")
    if rel_pos_h.shape != (2 * H - 1, d) or rel_pos_w.shape != (2 * W - 1, d):
        raise ValueError("relative position tables must be [2H-1, d] and [2W-1, d]")
    if table is None:
        table = rel_pos_table(rel_pos_h, rel_pos_w, qkv.dtype, qkv.device)
    rel_all = rel_pos_products(qkv, num_heads, table)
    if not rel_all.is_contiguous():
        rel_all = rel_all.contiguous()
    out = torch.empty((tokens, C), dtype=qkv.dtype, device=qkv.device)
    esz = qkv.element_size()
    with torch.cuda.device(qkv.device):
        with _Timed("attn_global", 4 * tokens * C * esz):
            _lib.check(lib.samq_attn_global(_ptr(qkv), None, _ptr(rel_all), _DTYPE_CODE[qkv.dtype], units, rel_all.shape[-1],
                                            H, W, num_heads, d, float(scale), _ptr(out), _ptr(status_word(qkv.device)), _stream()))
    return out


def attn_window14_supported(H: int, W: int, head_dim: int, dtype) -> bool:
    """Shapes ``samq_attn_window14`` is built for: SAM's 14 x 14 windows, head width 64 or 80."""
    return H == 14 and W == 14 and head_dim in (64, 80) and dtype in (torch.float16, torch.bfloat16)


def attn_window14(qkv: torch.Tensor, windows: int, num_heads: int, rel_pos_h: torch.Tensor, rel_pos_w: torch.Tensor,
                  scale: float, table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of 14 x 14 windows with the decomposed relative-position bias in one tensor-core
    kernel (``samq_attn_window14``): ``qkv`` [windows*196, 3C] -> [windows*196, C], same dtype.
    ``table`` is an optional cached ``rel_pos_table`` of the two [27, d] tables (56 rows)."""
    _require_cuda(qkv, "qkv")
    lib = _lib.load()
    tokens, three_c = qkv.shape
    C = three_c // 3
    d = C // num_heads
    if tokens != windows * 196 or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous [windows*196, 3C] tensor")
    if rel_pos_h.shape != (27, d) or rel_pos_w.shape != (27, d):
        raise ValueError("relative position tables must be [27, d]")
    if table is None:
        table = rel_pos_table(rel_pos_h, rel_pos_w, qkv.dtype, qkv.device)
    out = torch.empty((tokens, C), dtype=qkv.dtype, device=qkv.device)
    esz = qkv.element_size()
    with torch.cuda.device(qkv.device), _Timed("attn_window14", 4 * tokens * C * esz):
        _lib.check(lib.samq_attn_window14(_ptr(qkv), _ptr(table), table.shape[0], _DTYPE_CODE[qkv.dtype], windows, num_heads, d,
                                          float(scale), _ptr(out), _ptr(status_word(qkv.device)), _stream()))
    return out


def attn_windowed_supported(H: int, W: int, head_dim: int) -> bool:
    """Shapes ``samq_attn_windowed`` has a variant for."""
    L, J = H * W, 2 * H - 1 + 2 * W - 1
    return (L <= 16 and J <= 16 and head_dim in (16, 32, 64)) or (L <= 208 and J <= 56 and head_dim in (64, 80))


def attn_windowed(qkv: torch.Tensor, windows: int, H: int, W: int, num_heads: int, rel_pos_h: torch.Tensor,
                  rel_pos_w: torch.Tensor, scale: float, table: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Windowed attention with decomposed relative position bias in one kernel
    (``samq_attn_windowed``): ``qkv`` [windows*H*W, 3C] -> [windows*H*W, C], same dtype.
    ``table`` is an optional cached ``rel_pos_table`` of the two tables."""
    _require_cuda(qkv, "qkv")
    lib = _lib.load()
    tokens, three_c = qkv.shape
    C = three_c // 3
    d = C // num_heads
    if tokens != windows * H * W or not qkv.is_contiguous():
        raise ValueError("qkv must be a contiguous [windows*H*W, 3C] tensor")
    if rel_pos_h.shape != (2 * H - 1, d) or rel_pos_w.shape != (2 * W - 1, d):
        raise ValueError("relative position tables must be [2H-1, d] and [2W-1, d]")
    if table is None:
        table = rel_pos_table(rel_pos_h, rel_pos_w, qkv.dtype, qkv.device)
    out = torch.empty((tokens, C), dtype=qkv.dtype, device=qkv.device)
    with torch.cuda.device(qkv.device), _Timed("attn_window", tokens * 4 * C * qkv.element_size()):
        _lib.check(lib.samq_attn_windowed(_ptr(qkv), _DTYPE_CODE[qkv.dtype], windows, H, W, num_heads, d,
                                          _ptr(table), table.shape[0], float(scale), _ptr(out), _stream()))
    return out

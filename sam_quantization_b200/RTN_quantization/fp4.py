"""FP4Linear — a linear layer in microscaled 4-bit floating point, weights and activations.

The sibling of ``W8A8Linear`` for the tensor cores' 4-bit kinds, with the same ``from_float`` signature, so that
``replace_linear_with_target_and_quantize(model, FP4Linear, 4, [], weight_quant="nvfp4", act_quant="nvfp4")`` converts
a model (RTN_quantization/utils.py:33-61 walks it).  The reference's own 4-bit code (quant/qgemm) multiplies integers;
its model code has no 4-bit layer."""
from __future__ import annotations

import torch
from torch import nn

from .. import ops
from .._lib import ACT_GELU, ACT_NONE


class FP4Linear(nn.Module):
    """``y = x @ W^T + bias`` with both operands in ``weight_quant``: "nvfp4" (16 columns a scale, e4m3) or "mxfp4" (32
    columns, powers of two).  The weight is kept as codes and scales (``qcodes``, ``qscales`` and, for nvfp4, a power of
    two ``global_scale``) and the activation is quantized in every call, for nvfp4 under the power of two
    ``act_global_scale``: magnitudes beyond 2688 times it saturate and blocks below about 2^-6 times it lose resolution, so
    a layer whose activations are far from 1 is given its own (``calibrate``, ``set_fp4_act_scales``).
    ``output_global_scale`` is the same for the output, where ``quantize_output`` asks for it."""

    # callers that know this module may fuse the following GELU / residual add into the product
    supports_fused_epilogue = True
    act_global_scale = output_global_scale = 1.0          # of pickled modules that are older than these

    def __init__(self, in_features, out_features, bias=True, weight_quant="nvfp4", quantize_output=False):
        super().__init__()
        if weight_quant not in ops.FP4_FORMATS:
            raise ValueError(f"Invalid weight_quant: {weight_quant}")
        self.in_features, self.out_features = in_features, out_features
        self.weight_quant_name = self.act_quant_name = weight_quant
        self.quantize_output = bool(quantize_output)
        self.global_scale = self.act_global_scale = self.output_global_scale = 1.0
        self.compute_dtype = torch.float16
        self.register_buffer("qcodes", torch.zeros(out_features, (in_features + 31) // 32 * 16, dtype=torch.uint8))
        self.register_buffer("qscales", torch.zeros(ops.fp4_scale_shape(weight_quant, out_features, in_features), dtype=torch.uint8))
        self.register_buffer("bias", torch.zeros(out_features, dtype=torch.float16) if bias else None)

    @property
    def qweight(self) -> ops.Fp4Tensor:
        return ops.Fp4Tensor(self.qcodes, self.qscales, self.out_features, self.in_features, self.weight_quant_name, self.global_scale)

    @property
    def weight(self) -> torch.Tensor:
        """The dequantized weight, rounded to the layer dtype."""
        return self.qweight.dequantize(self.compute_dtype)

    @weight.setter
    def weight(self, value: torch.Tensor) -> None:
        """Assigning a float weight quantizes it."""
        self._quantize(value.detach().to(self.qcodes.device if self.qcodes.is_cuda else value.device))

    def _quantize(self, w: torch.Tensor) -> torch.Tensor:
        """Store ``w``; returns its fake-quantized value."""
        if tuple(w.shape) != (self.out_features, self.in_features):
            raise ValueError(f"weight must be [{self.out_features}, {self.in_features}]")
        g = ops.fp4_global_scale(float(w.abs().max())) if self.weight_quant_name == "nvfp4" else 1.0
        out = ops.quantize_fp4(w, self.weight_quant_name, global_scale=g, fake_quant=True)
        self.qcodes, self.qscales, self.global_scale = out["q"].codes, out["q"].scales, g
        self.compute_dtype = w.dtype
        return out["fq"]

    # -- checkpoints ---------------------------------------------------------------------------
    def get_extra_state(self):
        return {"kind": "FP4Linear", "in_features": self.in_features, "out_features": self.out_features,
                "weight_quant": self.weight_quant_name, "quantize_output": self.quantize_output,
                "global_scale": self.global_scale, "act_global_scale": self.act_global_scale,
                "output_global_scale": self.output_global_scale, "compute_dtype": str(self.compute_dtype).split(".")[-1]}

    def set_extra_state(self, state):
        self.quantize_output, self.global_scale = bool(state["quantize_output"]), float(state["global_scale"])
        self.act_global_scale = float(state.get("act_global_scale", 1.0))
        self.output_global_scale = float(state.get("output_global_scale", 1.0))
        self.compute_dtype = getattr(torch, state["compute_dtype"])

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        state, key = state_dict.get(prefix + "_extra_state"), prefix + "bias"
        if state is not None and state.get("weight_quant") != self.weight_quant_name:
            error_msgs.append(f"{prefix}: the checkpoint holds {state.get('weight_quant')}, the layer {self.weight_quant_name}")
            return
        if self.bias is not None and state_dict.get(key) is not None and state_dict[key].dtype != self.bias.dtype:
            self._buffers["bias"] = torch.empty_like(self.bias, dtype=state_dict[key].dtype)      # the bias keeps its dtype
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)

    # -- the layer -----------------------------------------------------------------------------
    def calibrate(self, act_absmax, output_absmax=None):
        """Choose the global scales of the activation and, with ``output_absmax``, of the output from their largest
        magnitudes in calibration.  mxfp4 has none and stays as it is.  Returns ``act_global_scale``."""
        if self.weight_quant_name == "nvfp4":
            self.act_global_scale = ops.fp4_global_scale(float(act_absmax))
            if output_absmax is not None:
                self.output_global_scale = ops.fp4_global_scale(float(output_absmax))
        return self.act_global_scale

    def act_quant(self, x):
        """The fake-quantized activation."""
        return ops.quantize_fp4(x, self.act_quant_name, global_scale=self.act_global_scale, fake_quant=True)["fq"]

    def output_quant(self, y):
        """The output as ``quantize_output`` asks for it."""
        if not self.quantize_output:
            return y
        return ops.quantize_fp4(y, self.act_quant_name, global_scale=self.output_global_scale, fake_quant=True)["fq"]

    @torch.no_grad()
    def forward(self, x, residual=None, activation=None, out_dtype=None):
        """As ``W8A8Linear.forward``: ``activation="gelu"`` and ``residual`` act in the product's epilogue, ``out_dtype``
        selects the stored type; with ``quantize_output`` the result is fake-quantized again."""
        y = ops.linear_fp4(x, self.qweight, bias=self.bias, residual=residual,
                           activation=ACT_GELU if activation == "gelu" else ACT_NONE, out_dtype=out_dtype,
                           x_global_scale=self.act_global_scale)
        return self.output_quant(y)

    @staticmethod
    def from_float(module, n_bits=4, weight_quant="nvfp4", act_quant=None, quantize_output=False, group_size=None):
        """The signature of ``W8A8Linear.from_float``.  Weight and activation share one 4-bit format, whose block is the
        group; the source module's weight is overwritten with its fake-quantized value.  The weight must live on a CUDA
        device."""
        assert isinstance(module, torch.nn.Linear)
        if weight_quant not in ops.FP4_FORMATS:
            raise ValueError(f"Invalid weight_quant: {weight_quant}")
        if act_quant not in (None, weight_quant):
            raise ValueError(f"Invalid act_quant: {act_quant} (the product takes two operands of one format, {weight_quant})")
        if n_bits != 4:
            raise ValueError(f"n_bits={n_bits}: {weight_quant} has 4")
        if group_size not in (None, ops.FP4_BLOCK[weight_quant]):
            raise ValueError(f"group_size={group_size}: {weight_quant} has blocks of {ops.FP4_BLOCK[weight_quant]}")
        new_module = FP4Linear(module.in_features, module.out_features, module.bias is not None, weight_quant, quantize_output)
        w = module.weight.data
        w.copy_(new_module._quantize(w))
        if module.bias is not None:
            new_module.bias = module.bias.data
        return new_module

    def __repr__(self):
        return (f"FP4Linear({self.in_features}, {self.out_features}, bias={self.bias is not None}, "
                f"weight_quant={self.weight_quant_name}, quantize_output={self.quantize_output})")


def set_fp4_act_scales(model, act_scales) -> int:
    """Give every ``FP4Linear`` of ``model`` that ``act_scales`` names the activation scale for its largest magnitude.
    ``act_scales``: {module name: per-channel largest |x|}, what ``get_act_scales_sam`` returns for the float model before
    it is converted.  Returns how many layers were set."""
    layers = dict(model.named_modules())
    named = [name for name in act_scales if isinstance(layers.get(name), FP4Linear)]
    for name in named:
        layers[name].calibrate(float(torch.as_tensor(act_scales[name]).max()))
    return len(named)

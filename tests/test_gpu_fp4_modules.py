"""FP4Linear and the norm in front of a quantized layer, as a model uses them."""
import copy

import pytest
import torch
from torch import nn

from sam_quantization_b200 import checkpoint, ops, sam_encoder
from sam_quantization_b200.RTN_quantization import (FP4Linear, W8A8Linear, get_act_scales_sam, replace_linear_with_target_and_quantize,
                                                    set_fp4_act_scales)

pytestmark = pytest.mark.gpu
FORMATS = ["mxfp4", "nvfp4"]


def _linear(K, N, dtype, dev, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    lin = nn.Linear(K, N, bias=bias).to(dtype)
    with torch.no_grad():
        lin.weight.copy_(torch.randn(N, K, generator=g) * 0.02)
        if bias:
            lin.bias.copy_(torch.randn(N, generator=g) * 0.1)
    return lin.to(dev)


def _reference(x, layer, residual=None, gelu=False):
    """The layer in 64 bits from the values its operands stand for, and the bound of its fp32 accumulation."""
    a = ops.quantize_fp4(x, layer.weight_quant_name, fake_quant=True)["q"].dequantize().double()
    w = layer.qweight.dequantize().double()
    y = a @ w.t() + (layer.bias.double() if layer.bias is not None else 0)
    bound = x.shape[-1] * 2.0 ** -23 * (a.abs() @ w.abs().t())
    if gelu:
        y, bound = torch.nn.functional.gelu(y), 1.2 * bound + 3e-7 + 2e-5 * y.abs()
    return (y if residual is None else y + residual.double()), bound


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 40, 2500])
def test_layer(cuda_device, fmt, dtype, M):
    lin = _linear(320, 264, dtype, cuda_device)
    before = lin.weight.detach().clone()
    layer = FP4Linear.from_float(lin, 4, weight_quant=fmt, act_quant=fmt)
    assert torch.equal(lin.weight, layer.weight) and not torch.equal(lin.weight, before)      # the source is fake-quantized
    # half a step of the largest spacing (2 between 4 and 6), under a block scale of at most max / 4 (mxfp4 saturates 8 to 6)
    assert (before.float() - layer.weight.float()).abs().max() <= before.float().abs().max() / 4 * 1.05
    g = torch.Generator().manual_seed(M)
    x, r = torch.randn(M, 320, generator=g).to(dtype).to(cuda_device), torch.randn(M, 264, generator=g).to(dtype).to(cuda_device)
    half = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    for kw in ({}, {"activation": "gelu"}, {"residual": r}, {"activation": "gelu", "residual": r}):
        y = layer(x, **kw)
        want, bound = _reference(x, layer, kw.get("residual"), "activation" in kw)
        assert y.dtype == dtype and ((y.double() - want).abs() <= bound + half * (want.abs() + bound) + 2.0 ** -25).all()
    assert layer(x.view(1, M, 320), out_dtype=torch.float32).shape == (1, M, 264)
    ops.check_status()


def test_refusals_and_assignment(cuda_device):
    lin = _linear(64, 48, torch.float16, cuda_device)
    for kw in ({"n_bits": 8}, {"weight_quant": "per_channel"}, {"act_quant": "per_token"}, {"group_size": 64}):
        with pytest.raises(ValueError):
            FP4Linear.from_float(lin, **{"n_bits": 4, **kw})
    layer = FP4Linear.from_float(lin, 4, weight_quant="nvfp4", act_quant="nvfp4", group_size=16, quantize_output=True)
    w = torch.randn(48, 64, device=cuda_device)
    layer.weight = w
    assert layer.compute_dtype == torch.float32 and (layer.weight - w).abs().max() <= w.abs().max() / 6 * 1.07
    with pytest.raises(ValueError):
        layer.weight = w[:, :32]
    x = torch.randn(3, 64, device=cuda_device).half()
    y = layer(x)
    assert torch.equal(y, layer.act_quant(ops.linear_fp4(x, layer.qweight, bias=layer.bias)))
    assert "nvfp4" in repr(layer)


@pytest.mark.parametrize("fmt", FORMATS)
def test_encoder_is_converted_saved_and_restored(cuda_device, fmt, tmp_path):
    kw = dict(img_size=64, embed_dim=64, depth=2, num_heads=4, window_size=2, global_attn_indexes=(1,), out_chans=32, device=cuda_device)
    model = sam_encoder.build_encoder("vit_b", seed=1, **kw)
    images = torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(0)).half().to(cuda_device)
    replace_linear_with_target_and_quantize(model, FP4Linear, 4, [], weight_quant=fmt, act_quant=fmt)
    assert all(isinstance(m, FP4Linear) for b in model.image_encoder.blocks for m in (b.attn.qkv, b.attn.proj, b.mlp.lin1, b.mlp.lin2))
    y = model(images)
    # the same network with every layer evaluated from the fake-quantized tensors in fp32
    twin = copy.deepcopy(model)

    class Twin(nn.Module):
        def __init__(self, layer):
            super().__init__()
            self.layer = layer

        def forward(self, x):
            a = self.layer.act_quant(x).float()
            return (a @ self.layer.qweight.dequantize().t() + self.layer.bias.float()).to(x.dtype)

    for b in twin.image_encoder.blocks:
        b.attn.qkv, b.attn.proj, b.mlp.lin1, b.mlp.lin2 = (Twin(m) for m in (b.attn.qkv, b.attn.proj, b.mlp.lin1, b.mlp.lin2))
    z = twin(images)
    assert torch.nn.functional.cosine_similarity(y.float().flatten(), z.float().flatten(), 0) > 0.99
    path = str(tmp_path / "fp4.pt")
    checkpoint.save_quantized(model, path)
    other = sam_encoder.build_encoder("vit_b", seed=2, **kw)
    checkpoint.load_quantized(other, path)
    assert torch.equal(other(images), y)
    wrong = FP4Linear(64, 192, True, "mxfp4" if fmt == "nvfp4" else "nvfp4").to(cuda_device)
    with pytest.raises(RuntimeError):
        wrong.load_state_dict(model.image_encoder.blocks[0].attn.qkv.state_dict())
    ops.check_status()


@pytest.mark.parametrize("M", [1, 300])
def test_a_block_of_a_rotated_network(cuda_device, M):
    """RMS norm with the residual's addition -> int8 linear with GELU -> 4-bit linear onto the residual stream, then the
    next norm: the pieces in the order a pre-norm block runs them, captured and replayed."""
    K, F = 256, 640
    up = W8A8Linear.from_float(_linear(K, F, torch.float16, cuda_device, 1), 8)
    down = FP4Linear.from_float(_linear(F, K, torch.float16, cuda_device, 2), 4, weight_quant="nvfp4", act_quant="nvfp4")
    g = torch.Generator().manual_seed(M)
    x, r = (torch.randn(M, K, generator=g).half().to(cuda_device) for _ in range(2))
    w = (1 + 0.2 * torch.randn(K, generator=g)).half().to(cuda_device)

    def block():
        h, stream = up.forward_rms_norm(x, w, 1e-6, residual=r, activation="gelu")
        return down(h, residual=stream), h, stream

    y, h, stream = block()
    assert torch.equal(stream, (x.float() + r.float()).half())
    # the first half against its definition: int8 codes of the norm, exact sums, erf GELU
    n = ops.rms_norm_quantize(x, w, 1e-6, residual=r)
    acc = (n["q"].double() * n["scale"].double()[:, None]) @ (up.qweight.double() * up.w_scale.double()[:, None]).t() + up.bias.double()
    want = torch.nn.functional.gelu(acc)
    assert ((h.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2e-5 * want.abs() + 1e-6).all()
    want, bound = _reference(h, down, stream)
    assert ((y.double() - want).abs() <= bound + 2.0 ** -11 * (want.abs() + bound) + 2.0 ** -25).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    graph.replay()
    assert torch.equal(out[0], y) and torch.equal(out[1], h)
    stream2 = r.clone()
    y2, s2 = up.forward_rms_norm(x, w, 1e-6, residual=stream2, residual_out=stream2, activation="gelu")
    assert s2 is stream2 and torch.equal(y2, h) and torch.equal(stream2, stream)
    with pytest.raises(ValueError):
        W8A8Linear.from_float(_linear(K, F, torch.float16, cuda_device), 8, act_quant="per_tensor").forward_rms_norm(x, w)
    ops.check_status()


@pytest.mark.parametrize("size", [1e-4, 1.0, 1e4])
def test_calibrated_activation_scale(cuda_device, size, tmp_path):
    lin = _linear(320, 264, torch.bfloat16, cuda_device)
    model = nn.Module()
    model.up = FP4Linear.from_float(lin, 4, weight_quant="nvfp4", act_quant="nvfp4", quantize_output=True)
    model.other = FP4Linear.from_float(_linear(320, 264, torch.bfloat16, cuda_device), 4, weight_quant="mxfp4", act_quant="mxfp4")
    x = (torch.randn(40, 320, generator=torch.Generator().manual_seed(1)) * size).to(torch.bfloat16).to(cuda_device)
    assert set_fp4_act_scales(model, {"up": x.abs().amax(0).float().cpu(), "other": torch.ones(320), "head": torch.ones(3)}) == 2
    layer = model.up
    g = ops.fp4_global_scale(float(x.abs().max()))
    assert layer.act_global_scale == g and model.other.act_global_scale == 1.0
    y = ops.linear_fp4(x, layer.qweight, bias=layer.bias, x_global_scale=g)
    layer.calibrate(x.abs().max(), y.abs().max())
    out = ops.fp4_global_scale(float(y.abs().max()))
    assert torch.equal(layer(x), ops.quantize_fp4(y, "nvfp4", global_scale=out, fake_quant=True)["fq"])
    a, w = layer.act_quant(x).double(), layer.qweight.dequantize().double()
    want = a @ w.t() + layer.bias.double()
    bound = 320 * 2.0 ** -23 * (a.abs() @ w.abs().t())
    assert ((y.double() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()
    assert ((a - x.double()).abs() <= x.abs().max().double() / 6 * 1.0625).all() and (a.count_nonzero() > 0.8 * a.numel())
    # the scales travel with the checkpoint; one without them has scales of 1
    torch.save(layer.state_dict(), str(tmp_path / "layer.pt"))
    other = FP4Linear(320, 264, True, "nvfp4").to(cuda_device)
    state = torch.load(str(tmp_path / "layer.pt"))
    other.load_state_dict(state)
    assert torch.equal(other(x), layer(x))
    for key in ("act_global_scale", "output_global_scale"):
        del state["_extra_state"][key]
    other.load_state_dict(state)
    assert other.act_global_scale == other.output_global_scale == 1.0
    ops.check_status()


def test_scales_of_a_float_encoder_reach_its_converted_layers(cuda_device):
    model = sam_encoder.build_encoder("vit_b", seed=1, img_size=64, embed_dim=64, depth=2, num_heads=4, window_size=2, global_attn_indexes=(1,),
                                      out_chans=32, device=cuda_device)
    images = torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(0)).half().to(cuda_device)
    scales = get_act_scales_sam(model, [images])
    replace_linear_with_target_and_quantize(model, FP4Linear, 4, [], weight_quant="nvfp4", act_quant="nvfp4")
    assert set_fp4_act_scales(model, scales) == len(scales) == 8
    layer = model.image_encoder.blocks[1].mlp.lin2
    assert layer.act_global_scale == ops.fp4_global_scale(float(scales["image_encoder.blocks.1.mlp.lin2"].max()))
    assert model(images).isfinite().all()
    ops.check_status()


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_layer_of_a_converted_encoder(cuda_device, fmt):
    """Each layer on what the encoder gives it (input, residual, activation, output type), against its definition."""
    model = sam_encoder.build_encoder("vit_b", seed=1, img_size=64, embed_dim=64, depth=2, num_heads=4, window_size=2, global_attn_indexes=(1,),
                                      out_chans=32, device=cuda_device)
    replace_linear_with_target_and_quantize(model, FP4Linear, 4, [], weight_quant=fmt, act_quant=fmt)
    seen, held = [], {}

    def before(layer, args, kw):
        held[layer] = (args[0].clone(), {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()})

    for layer in model.modules():
        if isinstance(layer, FP4Linear):
            layer.register_forward_pre_hook(before, with_kwargs=True)
            layer.register_forward_hook(lambda m, args, y: seen.append((m, *held[m], y.clone())))
    model(torch.rand(2, 3, 64, 64, generator=torch.Generator().manual_seed(0)).half().to(cuda_device))
    assert len(seen) == 8 and sum(kw.get("residual") is not None for _, _, kw, _ in seen) >= 2 and any(kw.get("activation") == "gelu" for _, _, kw, _ in seen)
    for layer, x, kw, y in seen:
        r = kw.get("residual")
        want, bound = _reference(x.reshape(-1, layer.in_features), layer, None if r is None else r.reshape(-1, layer.out_features), kw.get("activation") == "gelu")
        half = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[y.dtype]
        # the epilogue takes its bias in the output type: an fp16 bias under a bf16 output is off by half a step of it, up to 1.13
        # times that behind the GELU (its slope)
        if layer.bias.dtype != y.dtype:
            bound = bound + 1.13 * half * layer.bias.double().abs()
        # the alpha / bias step and the residual's addition: half a step of fp32 each
        assert ((y.reshape(want.shape).double() - want).abs() <= bound + (half + 2.0 ** -22) * (want.abs() + bound) + 2.0 ** -25).all()
    ops.check_status()

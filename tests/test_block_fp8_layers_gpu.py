"""Layers of block-scaled FP8 checkpoints, and the direct calls of the operators around them against the registered ops."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as ob

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


def _layer(device, k, parts, dtype, bias, seed=0):
    from vllm_amd.layers.linear import MergedColumnParallelLinear
    from vllm_amd.layers.quantization import get_quantization_config
    g = torch.Generator().manual_seed(seed)
    config = get_quantization_config("fp8").from_config(dict(quant_method="fp8", activation_scheme="dynamic", weight_block_size=[128, 128]))
    layer = MergedColumnParallelLinear(k, parts, bias=bias, quant_config=config, params_dtype=dtype, return_bias=False).to(device)
    w = (torch.randn((sum(parts), k), generator=g) * 60).clamp(-448, 448).to(FP8)
    s = torch.rand((ob.groups(sum(parts)), ob.groups(k)), generator=g) * 2e-4 + 1e-6
    layer.weight.weight_loader(layer.weight, w)
    layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, s)
    if bias:
        layer.bias.data.copy_(torch.randn(sum(parts), generator=g))
    layer.process_weights_after_loading()
    return layer, w, s


@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("k,parts", [(512, [256, 128, 128]), (400, [128, 144])])
@pytest.mark.parametrize("shape", [(1,), (37,), (2, 100), (300,)])
def test_layer(device, dtype, bias, k, parts, shape):
    layer, w, s = _layer(device, k, parts, dtype, bias)
    x = (torch.randn((*shape, k), generator=torch.Generator().manual_seed(1)) * 2).to(dtype)
    out = layer(x.to(device))
    assert out.shape == (*shape, sum(parts)) and out.dtype == dtype and out.is_contiguous()
    rows = x.reshape(-1, k)
    codes, scales = ob.group_quant(rows)      # the quantiser's bits are fixed, so that only the product's roundings remain
    want, magnitude = ob.block_scaled_mm(codes, w.t(), scales, s.t(), layer.bias.cpu() if bias else None)
    tol = want.abs() * torch.finfo(dtype).eps / 2 + magnitude * (128 + ob.groups(k) + 3) * 2.0 ** -23
    assert bool(((out.cpu().reshape(want.shape).double() - want).abs() <= tol).all())


def test_layer_keeps_a_hooked_quantiser_in_the_call(device):
    layer, _, _ = _layer(device, 256, [128, 128], torch.bfloat16, False)
    x = torch.randn((5, 256), device=device).to(torch.bfloat16)
    plain, seen = layer(x), []
    handle = layer.quant_method.block_linear.quant_fp8.register_forward_hook(lambda m, i, o: seen.append(o[0].shape))
    assert torch.equal(layer(x), plain) and seen == [(5, 256)]
    handle.remove()
    layer(x)
    assert len(seen) == 1


def test_layer_in_graphs(device):
    layer, _, _ = _layer(device, 512, [256, 256], torch.bfloat16, True)
    for m in (1, 70):
        x = torch.randn((m, 512), device=device).to(torch.bfloat16)
        layer(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        for step in range(3):
            x.add_(0.5)
            graph.replay()
            assert torch.equal(out.clone(), layer(x))
            torch.cuda.synchronize()


def _same(a, b):
    assert len(a) == len(b)
    for x, y in zip(a, b):
        assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
        assert torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8))


def test_direct_calls_equal_the_registered_ops(device):
    """The same bits, and an answer for every plain call."""
    from vllm_amd import _custom_ops as ops, _tuning
    f = ops._fast
    x = torch.randn((2, 9, 512), device=device).to(torch.bfloat16)
    rows, w, res = x.view(18, 512), torch.rand(512, device=device).to(torch.bfloat16), torch.randn((18, 512), device=device).to(torch.bfloat16)
    weight, sw = (torch.randn((272, 512), device=device) * 9).to(FP8).t(), torch.rand((3, 4), device=device).t()
    cache, pos = torch.rand((30, 64), device=device), torch.arange(18, device=device)
    head = w[:64]

    def calls():
        place = torch.empty_like(res)
        q, s = ops.scaled_fp8_group_quant(rows)
        yield ops.scaled_fp8_group_quant(x)
        yield ops.scaled_fp8_group_quant(rows[:, :384], output=torch.empty((18, 384), dtype=FP8, device=device))
        yield ops.silu_and_mul_group_quant(x)
        yield ops.rms_norm_group_quant(rows, w, 1e-5)
        yield (*ops.rms_norm_group_quant(rows, w, 1e-5, res, place), place)
        for a in (q, q.view(2, 9, 512)):
            yield (ops.block_scaled_mm(a, weight, s, sw, torch.float16, None), ops.block_scaled_mm(a, weight, s, sw, torch.bfloat16, res[0, :272].contiguous()))
        yield (ops.block_fp8_linear(x, weight, sw, torch.bfloat16, None),)
        yield ops.qk_norm_rope(rows, 4, 2, 64, 1e-6, head, head, cache, pos, False)

    direct = list(calls())
    with _tuning.override():      # (an override in force, even an empty one, sends every call through the registered op)
        for got, want in zip(direct, calls()):
            _same(got, want)
    assert f.group_quant(x, None) and f.silu_group_quant(x) and f.rms_norm_group_quant(rows, w, 1e-5, None, None)
    q, s = ops.scaled_fp8_group_quant(rows)
    assert f.block_mm(q, weight, s, sw, torch.float16, None) is not None and f.block_fp8_linear(x, weight, sw, torch.bfloat16, None) is not None
    assert f.qk_norm_rope(rows, 4, 2, 64, 1e-6, head, head, cache, pos, True, None, None) is not None


def test_bad_arguments_are_refused_by_both_routes(device):
    from vllm_amd import _custom_ops as ops
    x = torch.randn((6, 512), device=device).to(torch.bfloat16)
    q, s = ops.scaled_fp8_group_quant(x)
    w, sw = torch.zeros((256, 512), dtype=FP8, device=device).t(), torch.ones((4, 2), device=device)
    wide = torch.zeros((6, 1024), device=device, dtype=torch.bfloat16)
    cases = [
        (lambda: ops.scaled_fp8_group_quant(x.to(torch.float64)), "dtype"),
        (lambda: ops.scaled_fp8_group_quant(x.t()), "contiguous columns"),
        (lambda: ops.scaled_fp8_group_quant(x, output=torch.empty((6, 511), dtype=FP8, device=device)), "does not fit"),
        (lambda: ops.scaled_fp8_group_quant(x[:1].expand(6, 512)), "stride"),
        (lambda: ops.rms_norm_group_quant(x, x[0, :100], 1e-5), "weight"),
        (lambda: ops.rms_norm_group_quant(x, x[0], 1e-5, None, x), "residual_out"),
        (lambda: ops.rms_norm_group_quant(x, x[0], 1e-5, wide[:, :512]), "residual"),
        (lambda: ops.rms_norm_group_quant(x, x[0].float(), 1e-5), "weight"),
        (lambda: ops.block_scaled_mm(q, w, s[:, :3], sw, torch.bfloat16), "a_scales"),
        (lambda: ops.block_scaled_mm(q, w, s, sw.t(), torch.bfloat16), "b_scales"),
        (lambda: ops.block_scaled_mm(q, w, s, sw.double(), torch.bfloat16), "float32"),
        (lambda: ops.block_scaled_mm(q, w, s, sw, torch.float32), "float16 or bfloat16"),
        (lambda: ops.block_scaled_mm(q, w.contiguous(), s, sw, torch.bfloat16), "column-major"),
        (lambda: ops.block_scaled_mm(q[:, :256], w, s, sw, torch.bfloat16), "shape mismatch"),
        (lambda: ops.block_scaled_mm(q, w, s, sw, torch.bfloat16, x[0]), "bias"),
        (lambda: ops.block_scaled_mm(q[:, 8:264], w[:256], s[:, :2], sw[:2], torch.bfloat16), "aligned"),
        (lambda: ops.block_scaled_mm(q, w, s.cpu(), sw, torch.bfloat16), "GPU"),
        (lambda: ops.qk_norm_rope(x, 4, 4, 128, 1e-6, x[0, :128], x[0, :128], s, torch.arange(6, device=device)), "at least"),
        (lambda: ops.qk_norm_rope(x, 2, 1, 128, 1e-6, x[0, :128], x[0, :128], s, torch.arange(6, device=device).int()), "positions"),
        (lambda: ops.qk_norm_rope(x, 2, 1, 128, 1e-6, x[0, :64], x[0, :128], s, torch.arange(6, device=device)), "weights"),
        (lambda: ops.qk_norm_rope(x[:, 1:], 2, 1, 64, 1e-6, x[0, :64], x[0, :64], torch.rand((9, 64), device=device), torch.arange(6, device=device)), "aligned"),
    ]
    for call, text in cases:
        with pytest.raises(RuntimeError, match=text):
            call()
    with pytest.raises(NotImplementedError, match="float8_e4m3fn"):
        ops.block_scaled_mm(q.view(torch.uint8), w, s, sw, torch.bfloat16)


def test_linear_of_the_last_token_of_each_sequence(device):
    from vllm_amd import _custom_ops as ops
    x = torch.randn((3, 5, 256), device=device).to(torch.bfloat16)
    w = (torch.randn((144, 256), device=device) * 40).to(FP8).t()
    sw = torch.rand((2, 2), device=device)
    got = ops.block_fp8_linear(x[:, -1:], w, sw, torch.bfloat16, None)
    assert got.shape == (3, 1, 144)
    assert torch.equal(got, ops.block_fp8_linear(x[:, -1:].contiguous(), w, sw, torch.bfloat16, None))


def test_two_results_of_a_call_lie_apart(device):
    """They may be one allocation: each is a whole tensor of its own all the same."""
    from vllm_amd import _custom_ops as ops
    x = torch.randn((3, 260), device=device).to(torch.bfloat16)
    qkv, head = torch.randn((3, 5 * 24), device=device).to(torch.bfloat16), torch.ones(24, device=device, dtype=torch.bfloat16)
    pairs = [ops.scaled_fp8_group_quant(x), ops.silu_and_mul_group_quant(x), ops.rms_norm_group_quant(x, x[0], 1e-5),
             ops.qk_norm_rope(qkv, 3, 2, 24, 1e-6, head, head, torch.ones((4, 16), device=device), torch.tensor([0, 3, 1], device=device))]
    for a, b in pairs:
        assert a.is_contiguous() and not a.requires_grad and not b.requires_grad and a._version == 0 and b._version == 0
        one, other = a.clone(), b.clone()
        b.zero_()
        assert torch.equal(a.view(torch.uint8), one.view(torch.uint8)) and bool((b == 0).all()) and a._version == 0
        b.copy_(other)
        a.view(torch.uint8).zero_()
        assert torch.equal(b, other)
        kept = b
        del a, b
        assert torch.equal(kept, other)


def test_results_in_inference_mode_and_without_gradients(device):
    from vllm_amd import _custom_ops as ops
    x, w = torch.randn((5, 256), device=device).to(torch.bfloat16), (torch.randn((128, 256), device=device) * 40).to(FP8).t()
    sw = torch.rand((2, 1), device=device)
    want, scales = ops.scaled_fp8_group_quant(x)
    product = ops.block_scaled_mm(want, w, scales, sw, torch.bfloat16)
    for mode in (torch.inference_mode, torch.no_grad, torch.enable_grad):
        with mode():
            codes, s = ops.scaled_fp8_group_quant(x)
            assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(s, scales) and codes.is_inference() == s.is_inference()
            assert torch.equal(ops.block_scaled_mm(codes, w, s, sw, torch.bfloat16), product)
            assert torch.equal(s.clone().mul_(2), scales * 2)

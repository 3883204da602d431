"""Calls of the block-scaled FP8 operators as a model makes them: one row of a longer tensor, results that are kept, grown and saved apart."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("stride", [2048 * 4096, (1 << 22) + 16, 4096 + 8, 1])
def test_a_single_row_however_far_from_the_next(device, stride):
    """The last token of one long sequence is one row whose stride says nothing: past 4 MiB, odd, or shorter than the row.  By the direct call, the registered op
    and the op with an output whose stride says nothing either."""
    from vllm_amd import _custom_ops as ops, _tuning
    k, n = 4096, 272
    g = torch.Generator(device).manual_seed(5)
    codes = (torch.randn((1, k), device=device, generator=g) * 40).to(FP8)
    w = (torch.randn((n, k), device=device, generator=g) * 40).to(FP8).t()
    sa, sw = torch.rand((1, 32), device=device, generator=g), torch.rand((3, 32), device=device, generator=g).t()
    want = ops.block_scaled_mm(codes, w, sa, sw, torch.bfloat16)
    row = codes.as_strided((1, k), (stride, 1))
    assert torch.equal(ops.block_scaled_mm(row, w, sa, sw, torch.bfloat16), want)
    with _tuning.override():      # (through the registered op)
        assert torch.equal(ops.block_scaled_mm(row, w, sa, sw, torch.bfloat16), want)
    held = torch.zeros(n, dtype=torch.bfloat16, device=device)
    torch.ops.vllm_amd.block_scaled_mm(held.as_strided((1, n), (stride + 1, 1)), row, w, sa, sw, None)
    assert torch.equal(held[None], want)


def test_the_last_token_of_one_long_sequence(device):
    from vllm_amd import _custom_ops as ops
    g = torch.Generator(device).manual_seed(6)
    x = torch.randn((2048, 4096), device=device, generator=g).to(torch.bfloat16)
    w, sw = (torch.randn((128, 4096), device=device, generator=g) * 40).to(FP8).t(), torch.rand((32, 1), device=device, generator=g)
    codes, scales = ops.scaled_fp8_group_quant(x)
    want = ops.block_scaled_mm(codes[-1:].clone(), w, scales[-1:].clone(), sw, torch.bfloat16)
    last = codes.view(1, 2048, 4096)[:, -1]
    assert last.stride(0) > 1 << 22
    assert torch.equal(ops.block_scaled_mm(last, w, scales[-1:], sw, torch.bfloat16), want)
    assert torch.equal(ops.block_fp8_linear(x.view(1, 2048, 4096)[:, -1], w, sw, torch.bfloat16, None), want)


def _pairs(device):
    from vllm_amd import _custom_ops as ops
    g = torch.Generator(device).manual_seed(7)
    x = torch.randn((3, 256), device=device, generator=g).to(torch.bfloat16)
    qkv, head = torch.randn((3, 5 * 24), device=device, generator=g).to(torch.bfloat16), torch.ones(24, device=device, dtype=torch.bfloat16)
    cache, positions = torch.rand((4, 16), device=device, generator=g), torch.tensor([0, 3, 1], device=device)
    yield "quant", ops.scaled_fp8_group_quant(x)
    yield "silu", ops.silu_and_mul_group_quant(x)
    yield "norm", ops.rms_norm_group_quant(x, x[0].clone(), 1e-5)
    yield "rope", ops.qk_norm_rope(qkv, 3, 2, 24, 1e-6, head, head, cache, positions)


def test_each_result_of_a_call_has_a_storage_of_its_own(device):
    """Keeping or saving one does not keep the other, and one that grows in place does not run into the other."""
    for name, (a, b) in _pairs(device):
        for t in (a, b):
            assert t.untyped_storage().nbytes() == t.numel() * t.element_size() and t.storage_offset() == 0, name
        kept = b.clone()
        a.resize_((64, *a.shape[1:])).view(torch.uint8).fill_(255)
        assert torch.equal(b, kept), name


def _compiled(call):
    """`call` as a graph compiler runs it: traced, functionalised, its registered ops called one by one."""
    torch._dynamo.reset()
    return torch.compile(call, backend="aot_eager", fullgraph=True)


def test_traced_calls_give_the_same_bits(device):
    from vllm_amd import _custom_ops as ops
    from vllm_amd.layers.linear import LinearBase
    from vllm_amd.layers.quantization import get_quantization_config
    g = torch.Generator(device).manual_seed(8)
    x, res = (torch.randn((5, 384), device=device, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.rand(384, device=device, generator=g).to(torch.bfloat16)
    cache, positions = torch.rand((9, 64), device=device, generator=g), torch.tensor([0, 8, 3, 3, 1], device=device)
    config = get_quantization_config("fp8").from_config(dict(quant_method="fp8", activation_scheme="dynamic", weight_block_size=[128, 128]))
    layer = LinearBase(384, 144, quant_config=config, params_dtype=torch.bfloat16, return_bias=False).to(device)
    layer.weight.data.copy_((torch.randn((144, 384), device=device, generator=g) * 40).to(FP8))
    layer.weight_scale_inv.data.copy_(torch.rand((2, 3), device=device, generator=g))
    layer.process_weights_after_loading()

    def norm(x, held, place):
        return (*ops.rms_norm_group_quant(x, w, 1e-5, held, place), held, place)

    def norm_in_place(x, held):
        return (*ops.rms_norm_group_quant(x, w, 1e-5, held), held)

    def norm_twice_the_same(x, held):
        return (*ops.rms_norm_group_quant(x, w, 1e-5, held, held), held)

    def heads(x):
        return ops.qk_norm_rope(x, 4, 2, 64, 1e-6, w[:64], w[64:128], cache, positions)

    def chain(x):
        return (*ops.silu_and_mul_group_quant(x), *ops.scaled_fp8_group_quant(x), layer(x))
    with torch.no_grad():
        for call, args in ((norm, lambda: (x, res.clone(), torch.zeros_like(res))), (norm_in_place, lambda: (x, res.clone())),
                           (norm_twice_the_same, lambda: (x, res.clone())), (heads, lambda: (x,)), (chain, lambda: (x,))):
            want, got = call(*args()), _compiled(call)(*args())
            for a, b in zip(want, got, strict=True):
                assert a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8)), call.__name__


def test_results_on_top_of_what_they_are_made_of(device):
    """The sum with the residual over the input; both the same tensor; a single token's heads normed and rotated where they lie."""
    from vllm_amd import _custom_ops as ops
    g = torch.Generator(device).manual_seed(9)
    x, res = (torch.randn((70, 5120), device=device, generator=g).to(torch.float16) for _ in range(2))
    w = torch.rand(5120, device=device, generator=g).to(torch.float16)
    place = torch.empty_like(x)
    codes, scales = ops.rms_norm_group_quant(x, w, 1e-5, res, place)
    over = x.clone()
    codes2, scales2 = ops.rms_norm_group_quant(over, w, 1e-5, res, over)
    assert torch.equal(over, place) and torch.equal(codes2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scales2, scales)
    codes, scales = ops.rms_norm_group_quant(x, w, 1e-5, x.clone(), place)
    over = x.clone()
    codes2, scales2 = ops.rms_norm_group_quant(over, w, 1e-5, over)
    assert torch.equal(over, place) and torch.equal(codes2.view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scales2, scales)
    head, cache, position = w[:64], torch.rand((9, 64), device=device, generator=g), torch.tensor([7], device=device)
    qkv = x[:1].clone()      # 48 and 16 heads of 64, then values
    q, k = ops.qk_norm_rope(qkv, 48, 16, 64, 1e-6, head, head, cache, position)
    rest = qkv[:, 64 * 64:].clone()
    ops.qk_norm_rope(qkv, 48, 16, 64, 1e-6, head, head, cache, position, True, qkv[:, :48 * 64].view(1, 48, 64), qkv[:, 48 * 64:64 * 64].view(1, 16, 64))
    assert torch.equal(qkv[:, :48 * 64].view(q.shape), q) and torch.equal(qkv[:, 48 * 64:64 * 64].view(k.shape), k) and torch.equal(qkv[:, 64 * 64:], rest)

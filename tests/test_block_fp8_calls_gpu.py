"""Calls of the block-scaled FP8 operators as a model makes them: one row of a longer tensor."""
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

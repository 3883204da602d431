"""FP8 in groups and blocks of 128, and the head norms with rotation, from their definitions in 64 bits on the CPU (the group quantiser's codes in
fp32, which fixes them bit for bit).  Test infrastructure only."""
from __future__ import annotations

import torch

GROUP, FP8_MAX, LEAST = 128, 448.0, 1e-10
HALF_STEP, SMALLEST_HALF_STEP = 2.0 ** -4, 2.0 ** -10      # of e4m3: relative to a normal value; of the subnormal ones


def groups(n: int) -> int:
    return -(-n // GROUP)


def group_quant(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of [rows, columns] in fp32: the operator's result for any input type, bit for bit."""
    x = x.float()
    codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn)
    scales = torch.empty((x.shape[0], groups(x.shape[1])))
    for g in range(scales.shape[1]):
        part = x[:, g * GROUP:(g + 1) * GROUP]
        scales[:, g] = part.abs().amax(dim=1).clamp(min=LEAST) / FP8_MAX
        codes[:, g * GROUP:(g + 1) * GROUP] = (part / scales[:, g:g + 1]).to(torch.float8_e4m3fn)
    return codes, scales


def group_values(y: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(y over its group's scale, the scales) in 64 bits: what the codes round."""
    y = y.double()
    values, scales = torch.empty_like(y), torch.empty((y.shape[0], groups(y.shape[1])), dtype=torch.float64)
    for g in range(scales.shape[1]):
        part = y[:, g * GROUP:(g + 1) * GROUP]
        scales[:, g] = part.abs().amax(dim=1).clamp(min=LEAST) / FP8_MAX
        values[:, g * GROUP:(g + 1) * GROUP] = part / scales[:, g:g + 1]
    return values, scales


def silu_and_mul(x: torch.Tensor) -> torch.Tensor:
    gate, up = x.double().chunk(2, dim=-1)
    return gate / (1 + torch.exp(-gate)) * up


def rms_norm(x: torch.Tensor, weight: torch.Tensor, epsilon: float) -> torch.Tensor:
    x = x.double()
    return x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + epsilon) * weight.double()


def spread(scales: torch.Tensor, rows: int, columns: int, row_block: int, column_block: int) -> torch.Tensor:
    """Scales of blocks as one for each of rows x columns values."""
    r, c = torch.arange(rows) // row_block, torch.arange(columns) // column_block
    return scales.double()[r][:, c]


def block_scaled_mm(a, b, scale_a, scale_b, bias=None) -> tuple[torch.Tensor, torch.Tensor]:
    """The product in 64 bits, and the sum of its terms' magnitudes (which bounds what the order of a sum changes)."""
    (m, k), n = a.shape, b.shape[1]
    x = a.double() * spread(scale_a, m, k, 1, GROUP)
    y = b.double() * spread(scale_b, k, n, GROUP, GROUP)
    out = x @ y
    return (out if bias is None else out + bias.double()), x.abs() @ y.abs()


def qk_norm_rope(qkv, heads_q, heads_k, head_dim, epsilon, q_weight, k_weight, cache, positions, is_neox):
    tokens, rotary = qkv.shape[0], cache.shape[1]
    cos, sin = cache[positions].double()[:, None].chunk(2, dim=-1)
    outs, first = [], 0
    for heads, weight in ((heads_q, q_weight), (heads_k, k_weight)):
        y = rms_norm(qkv[:, first:first + heads * head_dim].reshape(tokens, heads, head_dim), weight, epsilon)
        first += heads * head_dim
        u_at = torch.arange(rotary // 2) * (1 if is_neox else 2)
        v_at = u_at + (rotary // 2 if is_neox else 1)
        u, v = y[..., u_at], y[..., v_at]
        y[..., u_at], y[..., v_at] = u * cos - v * sin, v * cos + u * sin
        outs.append(y)
    return tuple(outs)

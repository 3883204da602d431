"""Norms of query and key heads with the rotation by the token's position, against the oracle in 64 bits."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as ob

pytestmark = pytest.mark.gpu


def make(tokens, heads_q, heads_k, head_dim, rotary, dtype, cache_dtype, seed=0, extra=0, length=512):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn((tokens, (heads_q + 2 * heads_k) * head_dim + extra), generator=g) * 2).to(dtype)
    angle = torch.arange(length, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / max(rotary, 1))
    return dict(qkv=qkv, wq=(torch.randn(head_dim, generator=g) * 0.2 + 1).to(dtype), wk=(torch.randn(head_dim, generator=g) * 0.2 + 1).to(dtype),
                cache=torch.cat((angle.cos(), angle.sin()), 1).to(cache_dtype), positions=torch.randint(0, length, (tokens,), generator=g))


def call(c, heads_q, heads_k, head_dim, device, is_neox, epsilon=1e-6, **out):
    from vllm_amd import _custom_ops as ops
    d = {n: t.to(device) for n, t in c.items()}
    return ops.qk_norm_rope(d["qkv"], heads_q, heads_k, head_dim, epsilon, d["wq"], d["wk"], d["cache"], d["positions"], is_neox, **out)


def check(got, c, heads_q, heads_k, head_dim, is_neox, epsilon=1e-6):
    """One rounding to 16 bits (half a step of the value), and in fp32 a few roundings of the pair's magnitudes: the norm's sum over at most 512 squares (8 a lane, a
    tree over 64) and root, two products each."""
    want = ob.qk_norm_rope(c["qkv"], heads_q, heads_k, head_dim, epsilon, c["wq"], c["wk"], c["cache"], c["positions"], is_neox)
    for g, w in zip(got, want):
        assert g.shape == w.shape
        if w.numel() == 0:
            continue
        magnitude = w.abs().amax(dim=2, keepdim=True)
        tol = w.abs() * torch.finfo(g.dtype).eps / 2 + magnitude * 24 * 2.0 ** -24 + torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps
        d = (g.cpu().double() - w).abs()
        assert bool((d <= tol).all()), f"off by {(d - tol).max():.2e}"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("is_neox", [True, False])
@pytest.mark.parametrize("tokens,heads_q,heads_k,head_dim,rotary", [
    (1, 32, 8, 128, 128), (33, 28, 4, 128, 128), (3, 1, 1, 64, 64), (5, 16, 2, 256, 64), (7, 5, 5, 96, 96), (2, 3, 1, 80, 32),
    (4, 40, 8, 128, 32), (2, 2, 1, 512, 512), (6, 0, 3, 64, 16), (6, 3, 0, 64, 0), (1, 70, 10, 8, 0), (300, 8, 1, 192, 64)])
def test_qk_norm_rope(device, dtype, is_neox, tokens, heads_q, heads_k, head_dim, rotary):
    for cache_dtype in (torch.float32, dtype):
        c = make(tokens, heads_q, heads_k, head_dim, rotary, dtype, cache_dtype, seed=head_dim + tokens)
        check(call(c, heads_q, heads_k, head_dim, device, is_neox), c, heads_q, heads_k, head_dim, is_neox)


def test_rotary_dims_of_pairs(device):
    """Neighbours in pairs: rotated values that end inside a lane's eight."""
    for rotary in (2, 6, 10, 62):
        c = make(9, 4, 2, 64, rotary, torch.bfloat16, torch.float32, seed=rotary)
        check(call(c, 4, 2, 64, device, False), c, 4, 2, 64, False)


def test_wide_rows_and_padding(device):
    """qkv as a slice of wider rows, cos and sin as a slice; tokens without a position leave their rows as they are."""
    c = make(12, 4, 2, 128, 64, torch.bfloat16, torch.float32, seed=4, extra=72)
    c["positions"][3], c["positions"][7] = -1, 512
    qkv = c["qkv"].to(device)
    assert qkv.stride(0) % 8 == 0
    cache = torch.zeros((512, 100), device=device)
    cache[:, :64] = c["cache"].to(device)
    from vllm_amd import _custom_ops as ops
    q, k = torch.full((12, 4, 128), 7.0, dtype=torch.bfloat16, device=device), torch.full((12, 2, 128), 7.0, dtype=torch.bfloat16, device=device)
    held = qkv.clone()
    got = ops.qk_norm_rope(qkv, 4, 2, 128, 1e-6, c["wq"].to(device), c["wk"].to(device), cache[:, :64], c["positions"].to(device), True, q, k)
    assert got[0] is q and got[1] is k and torch.equal(qkv, held)
    live = [t for t in range(12) if t not in (3, 7)]
    for t in (3, 7):
        assert bool((q[t] == 7).all() and (k[t] == 7).all())
    part = dict(c, qkv=c["qkv"][live], positions=c["positions"][live])
    check((q[live], k[live]), part, 4, 2, 128, True)


def test_special_values_stay_in_their_head(device):
    c = make(3, 4, 2, 128, 128, torch.bfloat16, torch.float32, seed=5)
    c["qkv"][1, 128 + 5] = float("nan")
    c["qkv"][2, 4 * 128 + 9] = float("inf")
    c["qkv"][0, :128] = 0.0
    q, k = (t.cpu() for t in call(c, 4, 2, 128, device, True))
    assert bool(q[1, 1].isnan().all()) and bool(q[1, [0, 2, 3]].isfinite().all()) and bool(k[1].isfinite().all())
    assert bool((q[0, 0] == 0).all()) and bool(q[2].isfinite().all()) and bool(k[2, 1].isfinite().all()) and not bool(k[2, 0].isfinite().all())


def test_no_tokens(device):
    c = make(0, 4, 2, 128, 128, torch.bfloat16, torch.float32)
    q, k = call(c, 4, 2, 128, device, True)
    assert q.shape == (0, 4, 128) and k.shape == (0, 2, 128)


def test_in_a_graph_and_on_another_stream(device):
    from vllm_amd import _custom_ops as ops
    c = {n: t.to(device) for n, t in make(21, 8, 2, 128, 128, torch.bfloat16, torch.float32, seed=9).items()}

    def work():
        return ops.qk_norm_rope(c["qkv"], 8, 2, 128, 1e-6, c["wq"], c["wk"], c["cache"], c["positions"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = work()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, work()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for step in range(3):
        c["qkv"].mul_(1.0 + step)
        c["positions"].copy_((c["positions"] + 3) % 512)
        graph.replay()
        for a, b in zip([t.clone() for t in out], work()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_more_tokens_than_a_launch(device):
    from vllm_amd import _custom_ops as ops
    edge = 1 << 22
    qkv = torch.randn((edge + 3, 24), device=device, generator=torch.Generator(device).manual_seed(8)).to(torch.float16)
    angle = torch.rand((50, 8), device=device) * 6
    cache = torch.cat((angle[:, :4].cos(), angle[:, :4].sin()), 1)
    positions = torch.arange(edge + 3, device=device) % 50

    def work(rows):
        return ops.qk_norm_rope(qkv[rows], 1, 1, 8, 1e-6, qkv[0, :8].clone(), qkv[1, :8].clone(), cache, positions[rows].clone(), False)

    every = work(slice(None))
    for rows in (slice(0, 3), slice(edge - 3, edge + 3)):
        for a, b in zip(every, work(rows)):
            assert torch.equal(a[rows], b)

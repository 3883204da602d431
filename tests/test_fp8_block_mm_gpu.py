"""The FP8 product with a scale for each block of 128, against the oracle in 64 bits: the automatic choice and every kernel."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as ob

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
SHAPES = 7      # tile shapes
# blocks of 16 rows, n-tiles, steps ahead, wavefronts
ROWS = [(mb, j, ahead, waves) for mb in (1, 2, 3, 4) for j in (1, 2, 4) for ahead in (1, 2) for waves in (4, 8)
        if (mb + ahead * j) * waves < 40 and (waves == 4 or j == 1) and (j < 4 or ahead == 1)]


def make(m, k, n, dtype=torch.bfloat16, bias=False, seed=0):
    g = torch.Generator().manual_seed(seed * 1000 + m + k + n)
    kb, nb = ob.groups(k), ob.groups(n)
    return dict(a=(torch.randn((m, k), generator=g) * 60).clamp(-448, 448).to(FP8), w=(torch.randn((n, k), generator=g) * 60).clamp(-448, 448).to(FP8),
                sa=torch.rand((m, kb), generator=g) * 2e-2 + 1e-4, sw=torch.rand((nb, kb), generator=g) * 2e-4 + 1e-6, dtype=dtype,
                bias=torch.randn(n, generator=g).to(dtype) if bias else None)


def call(c, device):
    from vllm_amd import _custom_ops as ops
    d = {n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in c.items()}
    return ops.block_scaled_mm(d["a"], d["w"].t(), d["sa"].t().contiguous().t(), d["sw"].t(), c["dtype"], d["bias"])


def check(out, c, what=""):
    """One rounding to the output's type (half a step of the value), and sums in fp32: each of the K + K / 128 additions moves the sum by at most a step
    (2^-23: the matrix instruction's own additions need not round to nearest) of the terms' magnitudes."""
    want, magnitude = ob.block_scaled_mm(c["a"], c["w"].t(), c["sa"], c["sw"].t(), c["bias"])
    assert out.shape == want.shape and out.dtype == c["dtype"]
    steps = min(c["a"].shape[1], 128) + ob.groups(c["a"].shape[1]) + 3
    tol = want.abs() * torch.finfo(out.dtype).eps / 2 + magnitude * steps * 2.0 ** -23 + torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    d = (out.cpu().double() - want).abs()
    assert bool((d <= tol).all()), f"{what}: off by {(d - tol).max():.2e} of {want.abs().mean():.2e}"


SIZES = [(1, 16, 16), (1, 2048, 2048), (3, 128, 128), (16, 512, 272), (17, 4096, 1024), (33, 144, 400), (64, 2976, 1040), (65, 1024, 2048),
         (100, 7168, 576), (129, 256, 4112), (256, 1536, 1536), (257, 640, 272), (300, 80, 144), (515, 1040, 2064)]


@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True)])
def test_block_scaled_mm(device, m, k, n, dtype, bias):
    c = make(m, k, n, dtype, bias)
    check(call(c, device), c)


@pytest.mark.parametrize("shape", range(SHAPES))
@pytest.mark.parametrize("m,k,n", [(1, 16, 16), (70, 128, 144), (130, 272, 272), (257, 400, 528), (300, 1664, 1040), (64, 4096, 128), (520, 896, 1296)])
def test_every_tile_shape(device, shape, m, k, n):
    from vllm_amd import _tuning
    c = make(m, k, n, bias=m > 100)
    with _tuning.override(fp8_path=2, fp8_tile_cfg=shape + 1):
        check(call(c, device), c)


@pytest.mark.parametrize("mb,j,ahead,waves", ROWS)
@pytest.mark.parametrize("m,k,n", [(1, 16, 16), (15, 256, 48), (16, 1280, 144), (70, 2064, 208), (33, 3840, 64), (130, 4096, 80), (4, 9216, 128)])
def test_every_plan_for_few_rows(device, mb, j, ahead, waves, m, k, n):
    from vllm_amd import _tuning
    c = make(m, k, n, bias=m > 15)
    with _tuning.override(fp8_path=1, exp=[0] * 11 + [waves << 12 | ahead << 8 | mb << 4 | j]):
        check(call(c, device), c)


def _variants():
    yield "automatic", {}
    for shape in range(SHAPES):
        yield f"tile shape {shape}", dict(fp8_path=2, fp8_tile_cfg=shape + 1)
    for mb, j, ahead, waves in ROWS:
        yield f"rows {mb} x {j}, {ahead} ahead, {waves} wavefronts", dict(fp8_path=1, exp=[0] * 11 + [waves << 12 | ahead << 8 | mb << 4 | j])


def test_one_scale_each(device):
    """A one-hot row picks one row of the weight: its values times both scales, one rounding -- a wrong scale, block or row shows in full.  In every kernel."""
    from vllm_amd import _tuning
    m, k, n = 40, 1424, 656
    c = make(m, k, n)
    at = torch.randint(0, k, (m,), generator=torch.Generator().manual_seed(3))
    at[0], at[1], at[2] = 0, k - 1, 1408
    hot = torch.zeros((m, k))
    hot[torch.arange(m), at] = 1.0
    c["a"] = hot.to(FP8)
    kb, nb = at // 128, torch.arange(n) // 128
    scale = c["sa"][torch.arange(m), kb][:, None] * c["sw"][nb][:, kb].t()      # fp32, one rounding
    want = (c["w"].float().t()[at] * scale).to(torch.bfloat16)
    for name, fields in _variants():
        with _tuning.override(**fields):
            out = call(c, device).cpu()
        # the product with the scales is rounded to fp32 once more, or not: a tie of the last rounding may fall either way
        d = (out.double() - want.double()).abs()
        assert bool((d <= want.double().abs() * 2.0 ** -7).all()), name
        assert float((out != want).float().mean()) < 1e-3, name


@pytest.mark.parametrize("fill", [0x7f, 0x7e])
def test_what_lies_around_the_operands(device, fill):
    """Operands with wider rows, NaN (or the largest value) behind every row and behind the last one; scales as slices of NaN; an output with wider rows, whose
    surroundings stay."""
    from vllm_amd import _tuning
    for m, k, n in ((5, 272, 144), (70, 400, 272), (200, 1040, 528)):
        c = make(m, k, n, bias=True)
        kb, nb = ob.groups(k), ob.groups(n)
        a = torch.full((m + 300, k + 144), fill, dtype=torch.uint8, device=device).view(FP8)
        w = torch.full((n + 300, k + 144), fill, dtype=torch.uint8, device=device).view(FP8)
        a[:m, :k], w[:n, :k] = c["a"].to(device), c["w"].to(device)
        sa, sw = torch.full((m + 64, kb + 9), float("nan"), device=device), torch.full((nb + 3, kb + 9), float("nan"), device=device)
        sa[:m, :kb], sw[:nb, :kb] = c["sa"].to(device), c["sw"].to(device)
        for name, fields in _variants():
            for first, pitch in ((8, n + 24), (4, n + 12)):      # rows aligned to 16 bytes and to 8
                held = torch.full((m + 300, pitch), 3.0, dtype=torch.bfloat16, device=device)
                with _tuning.override(**fields):
                    torch.ops.vllm_amd.block_scaled_mm(held[:m, first:first + n], a[:m, :k], w[:n, :k].t(), sa[:m, :kb], sw[:nb, :kb].t(), c["bias"].to(device))
                check(held[:m, first:first + n], c, name)
                assert bool((held[m:] == 3).all() and (held[:, :first] == 3).all() and (held[:, first + n:] == 3).all()), name


def test_operands_past_four_gigabytes(device):
    """Rows 4 MiB apart: the last ones begin past 4 GiB, in the activations and in the weight."""
    from vllm_amd import _tuning
    pitch, rows = 1 << 22, 1040
    held = torch.zeros(rows * pitch, dtype=torch.uint8, device=device)
    for m, k, n in ((20, 400, 1040), (1040, 400, 144)):
        c = make(m, k, n)
        wide_w = n == rows
        far = held.view(FP8).view(rows, pitch)[:, :k]
        far.copy_((c["w"] if wide_w else c["a"]).to(device))
        near = (c["a"] if wide_w else c["w"]).to(device)
        from vllm_amd import _custom_ops as ops
        for name, fields in _variants():
            with _tuning.override(**fields):
                out = ops.block_scaled_mm(near if wide_w else far, far.t() if wide_w else near.t(), c["sa"].to(device), c["sw"].t().to(device), torch.bfloat16)
            check(out, c, name)


def test_special_values(device):
    """A NaN in a row is one in that row's results, one in a column in that column's; an infinite scale makes NaN of zeros and infinities of the rest."""
    from vllm_amd import _tuning
    m, k, n = 20, 512, 160
    c = make(m, k, n)
    c["a"].view(torch.uint8)[3, 77] = 0x7f
    c["w"].view(torch.uint8)[50, 300] = 0x7f
    c["sa"][7, 1] = float("inf")
    clean = torch.ones((m, n), dtype=torch.bool)
    clean[3], clean[:, 50], clean[7] = False, False, False
    for name, fields in _variants():
        with _tuning.override(**fields):
            out = call(c, device).cpu()
        assert bool(out[3].isnan().all()) and bool(out[:, 50].isnan().all()) and not bool(out[7].isfinite().any()), name
        assert bool(out[clean].isfinite().all()), name


def test_no_rows_and_many_dimensions(device):
    from vllm_amd import _custom_ops as ops
    c = make(0, 256, 128)
    assert call(c, device).shape == (0, 128)
    c = make(24, 256, 128)
    out = ops.block_scaled_mm(c["a"].to(device).view(2, 12, 256), c["w"].to(device).t(), c["sa"].to(device), c["sw"].t().to(device), torch.bfloat16)
    assert out.shape == (2, 12, 128)
    check(out.view(24, 128), c)


def test_in_graphs_and_on_streams(device):
    """Two captured graphs replayed on two streams at once, between eager calls: nothing is shared between calls."""
    cases = [make(9, 1024, 2048, seed=1), make(200, 1024, 2048, seed=2)]
    on = [{n: t.to(device) if isinstance(t, torch.Tensor) else t for n, t in c.items()} for c in cases]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in on:
        call(c, device)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(c, device))
        graphs.append(graph)
    for step in range(3):
        for c in on:
            c["sa"].mul_(0.75)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for c, out in zip(on, outs):
            assert torch.equal(out, call(c, device))


def test_a_block_of_operators(device):
    """RMSNorm with residual -> qkv -> head norms and rotation -> o -> RMSNorm -> gate/up -> SiLU-mul -> down, as a model runs them, against the same in 64 bits on
    the operators' own quantised values."""
    from vllm_amd import _custom_ops as ops
    g = torch.Generator().manual_seed(11)
    tokens, hidden, hq, hk, hd, ffn = 37, 512, 4, 2, 64, 1152
    x, res = (torch.randn((tokens, hidden), generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    norm = (torch.rand(hidden, generator=g) + 0.5).to(torch.bfloat16).to(device)
    qw = kw = torch.ones(hd, dtype=torch.bfloat16, device=device)
    angle = torch.arange(64)[:, None] * 0.1 ** torch.arange(hd // 2)
    cache, positions = torch.cat((angle.cos(), angle.sin()), 1).to(device), torch.arange(tokens, device=device)

    def weight(n, k):
        c = make(1, k, n, seed=n)
        return c["w"].to(device), c["sw"].to(device)

    def linear(q, s, wt):
        w, sw = wt
        out = ops.block_scaled_mm(q, w.t(), s, sw.t(), torch.bfloat16)
        check(out, dict(a=q.cpu(), w=w.cpu(), sa=s.cpu(), sw=sw.cpu(), bias=None, dtype=torch.bfloat16))
        return out

    q, s = ops.rms_norm_group_quant(x, norm, 1e-5, res)
    qkv = linear(q, s, weight((hq + 2 * hk) * hd, hidden))
    queries, keys = ops.qk_norm_rope(qkv, hq, hk, hd, 1e-6, qw, kw, cache, positions)
    want = ob.qk_norm_rope(qkv.cpu(), hq, hk, hd, 1e-6, qw.cpu(), kw.cpu(), cache.cpu(), positions.cpu(), True)
    for got, w in zip((queries, keys), want):
        assert float((got.cpu().double() - w).abs().max()) <= float(w.abs().max()) * 2.0 ** -8
    q, s = ops.scaled_fp8_group_quant(queries.view(tokens, -1))
    o = linear(q, s, weight(hidden, hq * hd))
    q, s = ops.rms_norm_group_quant(o, norm, 1e-5, res)
    gate_up = linear(q, s, weight(2 * ffn, hidden))
    q, s = ops.silu_and_mul_group_quant(gate_up)
    down = linear(q, s, weight(hidden, ffn))
    assert bool(down.isfinite().all())


def test_strides_of_single_rows_and_blocks_say_nothing(device):
    from vllm_amd import _custom_ops as ops
    w = (torch.randn((32, 256), device=device) * 40).to(torch.float8_e4m3fn).t()
    sw = torch.rand((2, 1), device=device)
    a = (torch.randn((7, 256), device=device) * 40).to(torch.float8_e4m3fn)
    sa = torch.rand((7, 2), device=device)
    far = sa[:1].as_strided((1, 2), (1 << 33, 1))
    assert torch.equal(ops.block_scaled_mm(a[:1], w, far, sw, torch.float16), ops.block_scaled_mm(a[:1], w, sa[:1], sw, torch.float16))
    one = sa.as_strided((7, 1), (2, 1 << 33))
    assert torch.equal(ops.block_scaled_mm(a[:, :128], w[:128], one, sw[:1].as_strided((1, 1), (1 << 33, 1)), torch.float16),
                       ops.block_scaled_mm(a[:, :128], w[:128], sa[:, :1], sw[:1], torch.float16))

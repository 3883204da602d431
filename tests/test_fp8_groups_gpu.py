"""FP8 quantisation in groups of 128 values, alone, behind SiLU-mul and behind RMSNorm, against the oracle."""
from __future__ import annotations

import pytest
import torch

from oracle import fp8_block as ob

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _bits(t):
    return t.cpu().view(torch.uint8)


def _randn(shape, seed, dtype, scale=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale
    x.view(-1)[::37] *= 30.0
    return x.to(dtype)


def check_codes(codes, scales, y64, rel):
    """Codes and scales of values that the kernel has to within `rel` of y64: a scale within that and its own rounding, a code within half a
    step of the value over the scale and what `rel` in both moves it."""
    value, scale = ob.group_values(y64)
    assert scales.shape == scale.shape
    d = (scales.cpu().double() - scale).abs()
    assert bool((d <= scale * (rel + 2.0 ** -23)).all()), f"scale off by {(d / scale).max():.2e}"
    d, v = (codes.cpu().double() - value).abs(), value.abs()
    bound = torch.maximum(v * ob.HALF_STEP, torch.tensor(ob.SMALLEST_HALF_STEP, dtype=torch.float64)) + v * (2 * rel + 2.0 ** -21)
    assert bool((d <= bound).all()), f"code off by {(d - bound).max():.2e}"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 130), (5, 127), (16, 512), (17, 4096), (33, 520), (2, 4104),
                                          (64, 1416), (4, 14336), (1000, 264)])
def test_group_quant_bits(device, dtype, rows, columns):
    from vllm_amd import _custom_ops as ops
    x = _randn((rows, columns), rows * 7 + columns, dtype)
    codes, scales = ops.scaled_fp8_group_quant(x.to(device))
    want, want_scales = ob.group_quant(x)
    assert codes.shape == x.shape and scales.shape == want_scales.shape and scales.stride(0) == 1
    assert torch.equal(scales.cpu(), want_scales)
    assert torch.equal(_bits(codes), _bits(want))


@pytest.mark.parametrize("dtype", TYPES)
def test_group_quant_strides_and_ranks(device, dtype):
    from vllm_amd import _custom_ops as ops
    wide = _randn((9, 1000), 3, dtype).to(device)
    for x in (wide[:, :512], wide[:, 8:648], wide[:, 3:131], wide[::3, :256], wide[:, :1], wide[4], wide[:8].view(2, 4, 1000)):
        codes, scales = ops.scaled_fp8_group_quant(x)
        flat = x.cpu().reshape(-1, x.shape[-1])
        want, want_scales = ob.group_quant(flat)
        assert codes.shape == x.shape
        assert torch.equal(scales.cpu(), want_scales) and torch.equal(_bits(codes.reshape(flat.shape)), _bits(want))
    # an output with wider rows: what lies between them stays
    held = torch.full((9, 1040), 5, dtype=torch.uint8, device=device)
    ops.scaled_fp8_group_quant(wide, output=held.view(torch.float8_e4m3fn)[:, 16:1016])
    assert torch.equal(held[:, 16:1016].cpu(), _bits(ob.group_quant(wide.cpu())[0]))
    assert bool((held[:, :16] == 5).all() and (held[:, 1016:] == 5).all())
    # scales in rows, through the registered op
    scales = torch.full((9, 12), -1.0, device=device)
    torch.ops.vllm_amd.scaled_fp8_group_quant(torch.empty((9, 1000), dtype=torch.float8_e4m3fn, device=device), wide, scales[:, 2:10])
    assert torch.equal(scales[:, 2:10].cpu(), ob.group_quant(wide.cpu())[1])
    assert bool((scales[:, :2] == -1).all() and (scales[:, 10:] == -1).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_group_quant_values_at_the_edges(device, dtype):
    from vllm_amd import _custom_ops as ops
    top = torch.finfo(dtype).max
    x = torch.randn((8, 512), generator=torch.Generator().manual_seed(1)).to(dtype)
    x[0] = 0.0
    x[0, 128:256] = -0.0
    x[1, :128] = torch.finfo(dtype).tiny
    x[2, :128] = top
    x[2, 130] = -top
    x[3, 5] = float("nan")
    x[4, 200] = float("inf")
    x[4, 201] = -float("inf")
    x[5, 300], x[5, 301] = float("nan"), float("inf")
    x[6] *= 1e-6
    codes, scales = ops.scaled_fp8_group_quant(x.to(device))
    want, want_scales = ob.group_quant(x)
    assert torch.equal(scales.cpu().isnan(), want_scales.isnan()) and bool(want_scales[3, 0].isnan())
    assert torch.equal(scales.cpu().nan_to_num(nan=-1.0), want_scales.nan_to_num(nan=-1.0))
    got, nan = codes.cpu().float(), want.float().isnan()
    assert torch.equal(got.isnan(), nan)
    assert torch.equal(_bits(codes)[~nan], _bits(want)[~nan])
    assert bool(nan[3, :128].all()) and not bool(nan[3, 128:].any()) and int(nan[4].sum()) == 2


def test_group_quant_empty(device):
    from vllm_amd import _custom_ops as ops
    for shape in ((0, 256), (3, 0), (0, 4, 128)):
        codes, scales = ops.scaled_fp8_group_quant(torch.empty(shape, dtype=torch.bfloat16, device=device))
        assert codes.shape == shape and scales.numel() == 0


# g / (1 + exp(-g)) * u in fp32 with the hardware's exponential and reciprocal: (|g| + 4) 2^-23 of the value (the exponential's argument is off by
# |g| 2^-23; a unit in the last place each for exponential and reciprocal, half for the sum and the two products); |g| is at most 40 here
SILU_REL = 44 * 2.0 ** -23


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("rows,d", [(1, 1), (1, 128), (7, 14336), (3, 130), (18, 520), (5, 127), (300, 256)])
def test_silu_and_mul_group_quant(device, dtype, rows, d):
    from vllm_amd import _custom_ops as ops
    x = (torch.randn((rows, 2 * d), generator=torch.Generator().manual_seed(d)) * 4).clamp(-40, 40).to(dtype)
    codes, scales = ops.silu_and_mul_group_quant(x.to(device))
    assert codes.shape == (rows, d)
    check_codes(codes, scales, ob.silu_and_mul(x), SILU_REL)
    # rows of a wider tensor, at an odd offset, and more than two dimensions
    wide = torch.zeros((rows, 2 * d + 5), dtype=dtype, device=device)
    wide[:, 3:3 + 2 * d] = x.to(device)
    again, again_scales = ops.silu_and_mul_group_quant(wide[:, 3:3 + 2 * d])
    assert torch.equal(_bits(again), _bits(codes)) and torch.equal(again_scales, scales)
    folded, _ = ops.silu_and_mul_group_quant(x.to(device).view(1, rows, 2 * d))
    assert folded.shape == (1, rows, d) and torch.equal(_bits(folded.view(rows, d)), _bits(codes))


def test_silu_and_mul_group_quant_infinities(device):
    from vllm_amd import _custom_ops as ops
    x = torch.randn((4, 512), generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    x[0, 3], x[1, 200], x[2, 7], x[3, 256 + 9] = float("inf"), -200.0, float("nan"), -float("inf")
    codes, scales = ops.silu_and_mul_group_quant(x.to(device))
    s = scales.cpu()
    assert s[0, 0] == float("inf") and bool(s[2, 0].isnan()) and s[3, 0] == float("inf")
    assert bool(s[1].isfinite().all()) and bool(s[:, 1].isfinite().all()) and codes.cpu().float()[1, 200] == 0
    got = codes.cpu().float()
    assert bool(got[2, :128].isnan().all()) and int(got[0].isnan().sum()) == 1 and int(got[3].isnan().sum()) == 1
    assert bool((got[0, :128].nan_to_num(nan=0.0) == 0).all())


# a sum of at most 65536 squares (64 a lane, a tree over 1024 lanes): (64 + 10) 2^-24, half of it in the root; root, division, two products and the sum with the residual
NORM_REL = 48 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("rows,hidden", [(1, 1), (3, 8), (1, 127), (2, 130), (5, 512), (32, 2048), (3, 2056), (32, 4096), (7, 5120),
                                         (2, 8192), (3, 14336), (2, 16392), (1, 65536), (2, 65535), (700, 1024)])
def test_rms_norm_group_quant(device, dtype, residual, rows, hidden):
    from vllm_amd import _custom_ops as ops
    x, w = _randn((rows, hidden), hidden, dtype), _randn((hidden,), 5, dtype, 0.1) + 1
    r = _randn((rows, hidden), 6, dtype, 3.0) if residual else None
    total = x.double() + (r.double() if residual else 0)
    want = ob.rms_norm(total, w, 1e-5)
    if not residual:
        codes, scales = ops.rms_norm_group_quant(x.to(device), w.to(device), 1e-5)
        check_codes(codes, scales, want, NORM_REL)
        return
    kept, given, place = r.to(device), r.to(device), torch.empty_like(r, device=device)
    codes, scales = ops.rms_norm_group_quant(x.to(device), w.to(device), 1e-5, kept, place)
    # the fp32 sum of two values of 16 bits is off by 2^-24 of itself: of the larger of them where they cancel, which the norm sees relative to the row
    check_codes(codes, scales, ob.rms_norm((x.float() + r.float()).double(), w, 1e-5), NORM_REL)
    assert torch.equal(kept.cpu(), r)
    assert torch.equal(place.cpu(), (x.float() + r.float()).to(dtype))
    codes2, scales2 = ops.rms_norm_group_quant(x.to(device), w.to(device), 1e-5, given)
    assert torch.equal(given, place) and torch.equal(_bits(codes2), _bits(codes)) and torch.equal(scales2, scales)


def test_rms_norm_group_quant_rows(device):
    """Rows of a wider tensor, at aligned and odd offsets; a row of zeros, of infinities and NaN."""
    from vllm_amd import _custom_ops as ops
    w = torch.ones(640, dtype=torch.bfloat16)
    wide = _randn((6, 1000), 8, torch.bfloat16).to(device)
    for first in (0, 8, 5):
        x = wide[:, first:first + 640]
        check_codes(*ops.rms_norm_group_quant(x, w.to(device), 1e-5), ob.rms_norm(x.cpu(), w, 1e-5), NORM_REL)
    x = _randn((4, 640), 9, torch.bfloat16)
    x[0], x[1, 70], x[2, 500] = 0.0, float("nan"), float("inf")
    codes, scales = ops.rms_norm_group_quant(x.to(device), w.to(device), 1e-5)
    got, s = codes.cpu().float(), scales.cpu()
    assert bool((got[0] == 0).all()) and bool((s[0] == torch.tensor(1e-10) / 448).all())
    assert bool(got[1].isnan().all()) and bool(s[1].isnan().all())
    assert int(got[2].isnan().sum()) == 128 and bool(s[2, 3].isnan()) and bool((got[2, :384] == 0).all())
    check_codes(codes[3:], scales[3:], ob.rms_norm(x[3:], w, 1e-5), NORM_REL)


def test_group_operators_in_a_graph(device):
    """Captured, and replayed between other work with new inputs: the results of the eager calls."""
    from vllm_amd import _custom_ops as ops
    x, gate = _randn((37, 1000), 1, torch.bfloat16).to(device), _randn((37, 512), 2, torch.bfloat16).to(device)
    w, res, out = torch.ones(1000, dtype=torch.bfloat16, device=device), _randn((37, 1000), 3, torch.bfloat16).to(device), None
    place = torch.empty_like(res)

    def work():
        return (*ops.scaled_fp8_group_quant(x), *ops.silu_and_mul_group_quant(gate), *ops.rms_norm_group_quant(x, w, 1e-5, res, place), place)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for seed in range(4):
        x.copy_(_randn((37, 1000), 10 + seed, torch.bfloat16))
        gate.copy_(_randn((37, 512), 20 + seed, torch.bfloat16))
        graph.replay()
        held = [t.clone() for t in out]
        for a, b in zip(held, work()):
            assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
        torch.cuda.synchronize()


def test_rows_one_stride_apart_in_more_dimensions(device):
    from vllm_amd import _custom_ops as ops
    held = _randn((3, 4, 1040), 5, torch.bfloat16).to(device)
    for x in (held[:, -1:, :512], held[:, :, :520], held[:, :1]):
        flat = x.reshape(-1, x.shape[-1])
        codes, scales = ops.scaled_fp8_group_quant(x)
        want, want_scales = ob.group_quant(flat.cpu())
        assert codes.shape == x.shape and torch.equal(scales.cpu(), want_scales) and torch.equal(_bits(codes.reshape(flat.shape)), _bits(want))
        for got, same in ((ops.silu_and_mul_group_quant(x), ops.silu_and_mul_group_quant(flat)),
                          (ops.rms_norm_group_quant(x, held[0, 0, :x.shape[-1]], 1e-6), ops.rms_norm_group_quant(flat, held[0, 0, :x.shape[-1]], 1e-6))):
            assert got[0].shape[:-1] == x.shape[:-1] and torch.equal(_bits(got[0]).reshape(_bits(same[0]).shape), _bits(same[0])) and torch.equal(got[1], same[1])
    with pytest.raises(RuntimeError, match="one stride apart"):
        ops.scaled_fp8_group_quant(held[:, :2, :512])


def test_scales_on_top_of_each_other_are_refused(device):
    x = _randn((4, 256), 6, torch.float16).to(device)
    codes = torch.empty((4, 256), dtype=torch.float8_e4m3fn, device=device)
    for scales in (torch.empty((1, 2), device=device).expand(4, 2), torch.empty(8, device=device).as_strided((4, 2), (1, 1)),
                   torch.empty(8, device=device).as_strided((4, 2), (1, 3))):
        with pytest.raises(RuntimeError, match="on top of each other"):
            torch.ops.vllm_amd.scaled_fp8_group_quant(codes, x, scales)


def test_norm_of_more_rows_than_a_launch(device):
    from vllm_amd import _custom_ops as ops
    edge = 1 << 21
    x = torch.randn((edge + 5, 8), device=device, generator=torch.Generator(device).manual_seed(7)).to(torch.bfloat16)
    residual, w = x.flip(0), x[0].clone()
    before = residual.clone()
    codes, scales = ops.rms_norm_group_quant(x, w, 1e-6, residual)
    for rows in (slice(0, 3), slice(edge - 3, edge + 5)):
        part = before[rows].clone()
        want, want_scales = ops.rms_norm_group_quant(x[rows].clone(), w, 1e-6, part)
        assert torch.equal(_bits(codes[rows]), _bits(want)) and torch.equal(scales[rows], want_scales) and torch.equal(residual[rows], part)

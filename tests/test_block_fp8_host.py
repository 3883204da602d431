"""CPU side of the block-scaled FP8 layers and of the operators around them: configuration, checkpoint loading, refusals of the ops and of the C ABI."""
from __future__ import annotations

import ctypes

import pytest
import torch

from oracle import fp8_block as ob
from vllm_amd import _custom_ops as ops
from vllm_amd import _lib
from vllm_amd.layers.linear import LinearBase, MergedColumnParallelLinear, QKVParallelLinear
from vllm_amd.layers.quantization import get_quantization_config

FP8 = torch.float8_e4m3fn


def config(**fields):
    return get_quantization_config("fp8").from_config({"quant_method": "fp8", "activation_scheme": "dynamic", "weight_block_size": [128, 128],
                                                       **fields})


# ------------------------------------------------------------------------------------------------ the oracle

def test_the_oracles_agree():
    """The group quantiser in fp32 and the values in 64 bits; the product in blocks and by the definition's own loops."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn((5, 300), generator=g)
    codes, scales = ob.group_quant(x)
    value, scale = ob.group_values(x)
    assert scales.shape == (5, 3) and float(((scales - scale) / scale).abs().max()) <= 2.0 ** -24
    half = torch.maximum(value.abs() * ob.HALF_STEP, torch.tensor(ob.SMALLEST_HALF_STEP, dtype=torch.float64))
    assert bool(((codes.double() - value).abs() <= half * (1 + 1e-6)).all()) and float(codes.float().abs().max()) == 448.0
    a, b = (torch.randn(s, generator=g).to(FP8) for s in ((3, 144), (144, 160)))
    sa, sb = torch.rand((3, 2), generator=g), torch.rand((2, 2), generator=g)
    out, _ = ob.block_scaled_mm(a, b, sa, sb)
    for m, n in ((0, 0), (2, 159), (1, 128), (1, 127)):
        want = sum(float(a[m, k]) * float(b[k, n]) * float(sa[m, k // 128]) * float(sb[k // 128, n // 128]) for k in range(144))
        assert abs(float(out[m, n]) - want) < 1e-10


def test_the_rotation_keeps_lengths_and_turns_pairs():
    qkv = torch.randn((4, 3 * 16), generator=torch.Generator().manual_seed(1)).double()
    angle = torch.arange(9)[:, None] * torch.tensor([1.0, 0.25])
    cache, one = torch.cat((angle.cos(), angle.sin()), 1).double(), torch.ones(16)
    q, _ = ob.qk_norm_rope(qkv, 1, 1, 16, 0.0, one, one, cache, torch.tensor([0, 1, 5, 8]), False)
    plain = ob.rms_norm(qkv[:, :16], one, 0.0)
    assert torch.allclose(q[0, 0], plain[0]) and torch.allclose(q[:, 0, 4:], plain[:, 4:])
    for t, pos in enumerate((0, 1, 5, 8)):
        for pair, frequency in ((0, 1.0), (1, 0.25)):
            z = complex(plain[t, 2 * pair], plain[t, 2 * pair + 1]) * complex(torch.cos(torch.tensor(pos * frequency)), torch.sin(torch.tensor(pos * frequency)))
            assert abs(complex(q[t, 0, 2 * pair], q[t, 0, 2 * pair + 1]) - z) < 1e-6


# ------------------------------------------------------------------------------------------------ configuration and loading

def test_config_refusals():
    assert config().weight_block_size == [128, 128]
    with pytest.raises(ValueError, match="two entries"):
        config(weight_block_size=[128])
    with pytest.raises(ValueError, match="dynamic"):
        config(activation_scheme="static")
    with pytest.raises(NotImplementedError, match="64, 128"):
        config(weight_block_size=[64, 128])
    with pytest.raises(ValueError, match="serialized"):
        get_quantization_config("fp8")(weight_block_size=[128, 128])


def test_weight_only_route_is_refused(monkeypatch):
    monkeypatch.setenv("VLLM_TEST_FORCE_FP8_MARLIN", "1")
    with pytest.raises(NotImplementedError, match="16-bit activations"):
        LinearBase(256, 128, quant_config=config())


def test_layer_sizes():
    with pytest.raises(ValueError, match="block_n"):
        MergedColumnParallelLinear(256, [192, 256], quant_config=config())
    with pytest.raises(ValueError, match="multiples of 16"):
        LinearBase(250, 128, quant_config=config())
    layer = MergedColumnParallelLinear(272, [256, 192], quant_config=config())      # the last part ends inside a block
    assert layer.weight_scale_inv.shape == (4, 3) and layer.weight.dtype == FP8 and layer.input_scale is None


def test_loading_parts_and_whole_tensors():
    g = torch.Generator().manual_seed(2)
    parts = [torch.rand((n, 2), generator=g) for n in (2, 1, 1)]      # 256, 128 and 128 output channels
    weights = [torch.randn((n * 128, 256), generator=g).to(FP8) for n in (2, 1, 1)]
    one = QKVParallelLinear(256, 64, 4, 2, quant_config=config())
    for shard, s, w in zip("qkv", parts, weights):
        one.weight_scale_inv.weight_loader(one.weight_scale_inv, s, shard)
        one.weight.weight_loader(one.weight, w, shard)
    whole = QKVParallelLinear(256, 64, 4, 2, quant_config=config())
    whole.weight_scale_inv.weight_loader(whole.weight_scale_inv, torch.cat(parts))
    whole.weight.weight_loader(whole.weight, torch.cat(weights))
    for layer in (one, whole):
        layer.process_weights_after_loading()
        assert torch.equal(layer.weight_scale_inv, torch.cat(parts).t()) and layer.weight.shape == (256, 512) and layer.weight.stride(0) == 1
        assert torch.equal(layer.weight.t().float(), torch.cat(weights).float())
    with pytest.raises(ValueError, match="does not fit"):
        bad = QKVParallelLinear(256, 64, 4, 2, quant_config=config())
        bad.weight_scale_inv.weight_loader(bad.weight_scale_inv, parts[0], "k")


# ------------------------------------------------------------------------------------------------ refusals of the ops

def test_no_cpu_fallback():
    x = torch.zeros((2, 256), dtype=torch.bfloat16)
    for call in (lambda: ops.scaled_fp8_group_quant(x), lambda: ops.silu_and_mul_group_quant(x),
                 lambda: ops.rms_norm_group_quant(x, x[0], 1e-5),
                 lambda: ops.block_scaled_mm(x.to(FP8), torch.zeros((128, 256), dtype=FP8).t(), torch.ones((2, 2)), torch.ones((2, 1)), torch.bfloat16),
                 lambda: ops.qk_norm_rope(x, 1, 1, 64, 1e-6, x[0, :64], x[0, :64], torch.zeros((4, 64)), torch.zeros(2, dtype=torch.int64))):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()
    for call in (ops.scaled_fp8_group_quant, ops.silu_and_mul_group_quant):
        with pytest.raises(NotImplementedError, match="group_size = 64"):
            call(x, group_size=64)
    with pytest.raises(RuntimeError, match="even"):
        ops.silu_and_mul_group_quant(x[:, :255])


def test_the_ops_have_shapes_without_a_gpu():
    """Fake tensors: what a graph compiler sees."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty((6, 300), dtype=torch.bfloat16, device="cuda")
        q, s = ops.scaled_fp8_group_quant(x)
        assert q.shape == (6, 300) and s.shape == (6, 3) and s.stride() == (1, 6)
        q, s = ops.silu_and_mul_group_quant(x)
        assert q.shape == (6, 150) and s.shape == (6, 2)
        q, s = ops.rms_norm_group_quant(x, x[0], 1e-5, x, x)
        assert q.shape == (6, 300) and s.shape == (6, 3)
        a = torch.empty((2, 3, 256), dtype=FP8, device="cuda")
        out = ops.block_scaled_mm(a, torch.empty((128, 256), dtype=FP8, device="cuda").t(), torch.empty((6, 2), device="cuda"),
                                  torch.empty((2, 1), device="cuda"), torch.float16)
        assert out.shape == (2, 3, 128) and out.dtype == torch.float16
        q, k = ops.qk_norm_rope(x, 3, 1, 64, 1e-6, x[0, :64], x[0, :64], torch.empty((9, 64), device="cuda"),
                                torch.empty(6, dtype=torch.int64, device="cuda"))
        assert q.shape == (6, 3, 64) and k.shape == (6, 1, 64)


# ------------------------------------------------------------------------------------------------ refusals of the C ABI (no launch, made-up addresses)

P = 1 << 20      # an aligned address that is never followed


def refused(name, args, status, text):
    lib = _lib.load()
    rc = getattr(lib, name)(*args)
    assert rc == status, (name, args, rc)
    assert text in lib.vaq_last_error().decode(), lib.vaq_last_error()


def with_(base: dict, **fields):
    assert set(fields) <= set(base)
    return list({**base, **fields}.values())


BAD, NOT_BUILT = _lib.VAQ_ERR_INVALID_ARG, _lib.VAQ_ERR_UNSUPPORTED


def test_group_quant_refusals():
    base = dict(i=P, dtype=_lib.VAQ_BF16, ld=256, out=P, ldo=256, s=P, sr=1, sg=4, rows=4, hidden=256, stream=None)
    for fields, text in ((dict(dtype=9), "in_dtype"), (dict(i=None), "null"), (dict(out=None), "null"), (dict(s=None), "null"), (dict(ld=255), "stride"),
                         (dict(ldo=200), "stride"), (dict(i=P + 1), "aligned"), (dict(s=P + 2), "aligned"), (dict(rows=-1), "rows"), (dict(hidden=1 << 31), "hidden")):
        refused("vaq_fp8_group_quant", with_(base, **fields), BAD, text)
    assert _lib.load().vaq_fp8_group_quant(*with_(base, rows=0, i=None, out=None, s=None)) == 0
    refused("vaq_silu_and_mul_fp8_group_quant", with_(base, ld=511), BAD, "stride")
    refused("vaq_silu_and_mul_fp8_group_quant", with_(base, ld=512, dtype=_lib.VAQ_F32), BAD, "dtype")


def test_norm_refusals():
    base = dict(out=P, s=P, sr=1, sg=4, i=P, ld=256, w=P, eps=1e-5, res=P, place=P, dtype=_lib.VAQ_F16, tokens=4, hidden=256, stream=None)
    for fields, text in ((dict(w=None), "null"), (dict(res=None), "null"), (dict(place=None), "null"), (dict(dtype=_lib.VAQ_F32), "dtype"), (dict(ld=8), "stride"),
                         (dict(w=P + 1), "aligned")):
        refused("vaq_rms_norm_fp8_group_quant", with_(base, **fields), BAD, text)
    refused("vaq_rms_norm_fp8_group_quant", with_(base, hidden=65537, ld=70000), NOT_BUILT, "65537")


def test_mm_refusals():
    base = dict(a=P, lda=256, b=P, ldb=256, sa=P, sar=1, sab=8, sb=P, sbk=1, sbn=2, bias=None, out=P, ldc=128, dtype=_lib.VAQ_BF16, m=8, n=128, k=256, stream=None)
    for fields, text in ((dict(a=None), "null"), (dict(b=None), "null"), (dict(sa=None), "null"), (dict(sb=None), "null"), (dict(out=None), "null"),
                         (dict(dtype=_lib.VAQ_F32), "out_dtype"), (dict(k=250), "multiples of 16"), (dict(n=120), "multiples of 16"), (dict(k=0), "K = 0"),
                         (dict(lda=248), "strides"), (dict(lda=240), "strides"), (dict(ldb=240), "strides"), (dict(ldc=124), "strides"), (dict(ldc=130), "strides"),
                         (dict(a=P + 8), "aligned"), (dict(out=P + 4), "aligned"), (dict(sa=P + 1), "aligned"), (dict(sar=-1), "negative"), (dict(m=1 << 31), "M = ")):
        refused("vaq_fp8_block_scaled_mm", with_(base, **fields), BAD, text)
    for fields, text in ((dict(lda=(1 << 22) + 16), "4 MiB"), (dict(ldb=1 << 23), "4 MiB"), (dict(sar=1 << 21), "2 GiB"), (dict(sab=1 << 29), "2 GiB"),
                         (dict(sbk=1 << 29), "2 GiB")):
        refused("vaq_fp8_block_scaled_mm", with_(base, **fields), NOT_BUILT, text)
    assert _lib.load().vaq_fp8_block_scaled_mm(*with_(base, m=0, a=None, sa=None, out=None)) == 0


def test_mm_plans_that_are_not_built():
    base = dict(a=P, lda=256, b=P, ldb=256, sa=P, sar=1, sab=8, sb=P, sbk=1, sbn=2, bias=None, out=P, ldc=128, dtype=_lib.VAQ_BF16, m=8, n=128, k=256, stream=None)
    t = _lib.VaqTuning()
    t.fp8_path = 2
    refused("vaq_fp8_block_scaled_mm_tuned", [*base.values(), ctypes.byref(t)], NOT_BUILT, "tile shape")
    t.fp8_path, t.exp[11] = 1, 4 << 12 | 2 << 8 | 4 << 4 | 4
    refused("vaq_fp8_block_scaled_mm_tuned", [*base.values(), ctypes.byref(t)], NOT_BUILT, "few rows")


def test_mm_of_more_than_a_launch():
    base = dict(a=P, lda=16, b=P, ldb=16, sa=P, sar=1, sab=8, sb=P, sbk=1, sbn=2, bias=None, out=P, ldc=16, dtype=_lib.VAQ_BF16, m=(1 << 31) - 16, n=16, k=16, stream=None)
    refused("vaq_fp8_block_scaled_mm", base.values(), NOT_BUILT, "threads")
    t = _lib.VaqTuning()
    t.fp8_path, t.fp8_tile_cfg = 2, 1
    refused("vaq_fp8_block_scaled_mm_tuned", [*with_(base, m=1 << 29), ctypes.byref(t)], NOT_BUILT, "threads")


def test_rope_refusals():
    base = dict(qkv=P, ld=768, q=P, k=P, hq=4, hk=1, d=128, eps=1e-6, wq=P, wk=P, cs=P, cs_dtype=_lib.VAQ_F32, cs_ld=128, cs_rows=9, rotary=128, inter=0, pos=P,
                dtype=_lib.VAQ_BF16, tokens=3, stream=None)
    for fields, text in ((dict(dtype=_lib.VAQ_F32), "dtype"), (dict(cs_dtype=_lib.VAQ_F16), "fp32"), (dict(hq=0, hk=0), "heads"), (dict(hq=-1), "heads"),
                         (dict(rotary=130), "rotary_dim"), (dict(rotary=31), "rotary_dim"), (dict(qkv=None), "null"), (dict(q=None), "null"), (dict(pos=None), "null"),
                         (dict(cs=None), "null"), (dict(ld=632), "stride"), (dict(ld=770), "aligned"), (dict(qkv=P + 2), "aligned"), (dict(wq=P + 8), "aligned"),
                         (dict(cs_ld=64), "cos_sin")):
        refused("vaq_qk_norm_rope", with_(base, **fields), BAD, text)
    for fields, text in ((dict(d=100, rotary=16, ld=1000), "head_dim"), (dict(d=520, ld=5200), "head_dim"), (dict(rotary=24), "rotary_dim")):
        refused("vaq_qk_norm_rope", with_(base, **fields), NOT_BUILT, text)
    assert _lib.load().vaq_qk_norm_rope(*with_(base, tokens=0, qkv=None)) == 0


# ------------------------------------------------------------------------------------------------ plans of the product

def test_prices_are_those_of_the_fit_and_choose_well():
    """profiles/plan_prices/fp8_block.py restates the prices: the library's plan is the cheapest of its, at its price; on the recorded times the choice is near the best."""
    import importlib.util
    import os

    import numpy as np
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "profiles", "plan_prices", "fp8_block.py")
    spec = importlib.util.spec_from_file_location("fp8_block_prices", path)
    f = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(f)
    few, tiles = f.tables()
    assert [len(r) for r in few.values()] == [9] * 4 and [len(r) for r in tiles] == [8] * 7
    _, by_problem = f.load()
    problems = list(by_problem)[:300]
    assert f.choice({p: by_problem[p] for p in problems}, few, tiles).mean() < 1.03
    lib, plan = _lib.load(), (ctypes.c_double * 6)()
    for m, k, n in problems[:100]:
        assert lib.vaq_fp8_block_plan(m, n, k, plan) == 0
        mb, j, ahead, waves, shape = map(int, plan[:5])
        name = f"r{mb}.{j}.{ahead}.{waves}" if mb else f"t{shape}"
        at = [np.array([float(x)]) for x in (m, k, n)]
        assert float(f.price(name, few, tiles, *at)[0]) == pytest.approx(plan[5], rel=1e-9)
        for other in by_problem[m, k, n]:
            assert float(f.price(other, few, tiles, *at)[0]) >= plan[5] * (1 - 1e-9)


def test_every_plan_in_reach_is_built():
    """The cheapest plan of small, large and odd problems is one that the launch takes (a plan that is not built would be refused at its call)."""
    lib, plan = _lib.load(), (ctypes.c_double * 6)()
    for m in (1, 15, 17, 48, 64, 100, 333, 1024, 1025, 8192):
        for k in (16, 512, 2976, 14336, 131072):
            for n in (16, 144, 4096, 28672, 262144):
                assert lib.vaq_fp8_block_plan(m, n, k, plan) == 0 and plan[5] > 0
                mb, j, ahead, waves, shape = map(int, plan[:5])
                assert (mb == 0 and 0 <= shape < 7) or ((mb + ahead * j) * waves < 40 and j in (1, 2, 4) and (waves == 4 or j == 1) and (j < 4 or ahead == 1))

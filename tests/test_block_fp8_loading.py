"""Block-scaled FP8 checkpoints that do not hold what their layers need, and modules that they leave unquantised."""
from __future__ import annotations

import pytest
import torch

from vllm_amd.layers.linear import LinearBase, MergedColumnParallelLinear, QKVParallelLinear, UnquantizedLinearMethod
from vllm_amd.layers.quantization import get_quantization_config

FP8 = torch.float8_e4m3fn


def config(**fields):
    return get_quantization_config("fp8").from_config({"quant_method": "fp8", "activation_scheme": "dynamic", "weight_block_size": [128, 128],
                                                       **fields})


def test_scales_that_the_checkpoint_does_not_hold():
    """None of a layer's, those of one part of a fused layer, or a single one that is the initial value: each is named when loading ends, instead of infinities later."""
    layer = LinearBase(256, 128, quant_config=config(), prefix="model.layers.0.o_proj")
    layer.weight.weight_loader(layer.weight, torch.zeros((128, 256), dtype=FP8))
    with pytest.raises(ValueError, match=r"model\.layers\.0\.o_proj.*2 of 2 .*weight_scale_inv"):
        layer.process_weights_after_loading()
    layer.weight_scale_inv.weight_loader(layer.weight_scale_inv, torch.ones((1, 2)))
    layer.process_weights_after_loading()

    fused = QKVParallelLinear(256, 64, 4, 2, quant_config=config())
    for shard, blocks in (("q", 2), ("v", 1)):
        fused.weight_scale_inv.weight_loader(fused.weight_scale_inv, torch.ones((blocks, 2)), shard)
    with pytest.raises(ValueError, match="2 of 8 .*weight_scale_inv"):
        fused.process_weights_after_loading()
    fused.weight_scale_inv.weight_loader(fused.weight_scale_inv, torch.zeros((1, 2)), "k")      # (a scale of zero is a scale)
    fused.process_weights_after_loading()
    assert fused.weight_scale_inv.shape == (2, 4) and float(fused.weight_scale_inv.sum()) == 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, torch.float8_e5m2])
def test_weights_of_another_type_are_not_rounded_to_fp8(dtype):
    """A checkpoint whose weight is not FP8 has no scales that fit it: whole, as a part, and as a whole tensor of a fused layer."""
    layer = LinearBase(256, 128, quant_config=config())
    with pytest.raises(ValueError, match=str(dtype)):
        layer.weight.weight_loader(layer.weight, torch.zeros((128, 256), dtype=dtype))
    fused = MergedColumnParallelLinear(256, [128, 128], quant_config=config())
    with pytest.raises(ValueError, match=str(dtype)):
        fused.weight.weight_loader(fused.weight, torch.zeros((128, 256), dtype=dtype), 1)
    with pytest.raises(ValueError, match=str(dtype)):
        fused.weight.weight_loader(fused.weight, torch.zeros((256, 256), dtype=dtype))
    fused.weight.weight_loader(fused.weight, torch.ones((128, 256), dtype=FP8), 1)
    assert bool((fused.weight.data[128:].float() == 1).all())


def test_modules_to_not_convert():
    """The key under which block-scaled checkpoints name what they leave in 16 bits, alone and beside ``ignored_layers``."""
    for fields in (dict(modules_to_not_convert=["lm_head", "model.layers.3"]), dict(ignored_layers=["lm_head"], modules_to_not_convert=["model.layers.3"]),
                   dict(ignored_layers=["lm_head", "model.layers.3"], modules_to_not_convert=None)):
        c = config(**fields)
        for prefix, plain in (("lm_head", True), ("model.layers.3.mlp.gate", True), ("model.layers.30.mlp.gate", False), ("model.layers.2.o_proj", False)):
            layer = LinearBase(256, 128, quant_config=c, prefix=prefix)
            assert isinstance(layer.quant_method, UnquantizedLinearMethod) == plain, (fields, prefix)
    assert config().ignored_layers == []

"""apply_quantization_config(keep_packed=True) over models in which not every weight can stay packed"""
import warnings

import pytest
import torch

from compressed_tensors_amd import CompressedLinear
from compressed_tensors_amd.config import QuantizationStatus
from compressed_tensors_amd.quantization import (QuantizationArgs, QuantizationConfig, QuantizationScheme,
                                                 apply_quantization_config)


def model():
    return torch.nn.ModuleDict({name: torch.nn.Linear(256, 32) for name in ("first", "second", "third")})


def config(**second):
    four = dict(num_bits=4, type="int", symmetric=True, strategy="group", group_size=64)
    groups = {"a": QuantizationScheme(targets=["re:(first|third)"], weights=QuantizationArgs(**four)),
              "b": QuantizationScheme(targets=["re:second"], weights=QuantizationArgs(**{**four, **second}))}
    return QuantizationConfig(config_groups=groups, format="pack-quantized", quantization_status="compressed")


@pytest.mark.parametrize("second", [dict(num_bits=8), dict(group_size=16), dict(actorder="group")])
def test_weights_that_cannot_stay_packed_are_decompressed_at_their_first_call(second):
    """whatever comes before them in the model, and after"""
    net = model()
    with pytest.warns(UserWarning, match="second"):
        apply_quantization_config(net, config(**second), run_compressed=True, keep_packed=True)
    assert all(type(m) is CompressedLinear and hasattr(m, "weight_packed") for m in net.values())
    assert [m.keep_packed for m in net.values()] == [True, False, True]
    assert all(m.quantization_status == QuantizationStatus.COMPRESSED for m in net.values())


def test_weights_that_can_stay_packed_all_do():
    net = model()
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        apply_quantization_config(net, config(), run_compressed=True, keep_packed=True)
    assert all(m.keep_packed for m in net.values())

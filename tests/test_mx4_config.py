"""MXFP4 configs: what the method does not implement is refused by name, and a model with such a config is none of
its own."""
import logging

import pytest

from sglite_amd.model_config import load_quantization_config
from sglite_amd.quantization import MXFP4Config

OTHERS = [{"modules_to_not_convert": ["model.layers.*.self_attn", "lm_head"]}, {"dequantize": True},
          {"kv_cache_scheme": {"num_bits": 8}}, {"weight_bits": 8}]


@pytest.mark.parametrize("other", OTHERS)
def test_what_it_does_not_implement(other, tmp_path, caplog):
    config = {"quant_method": "mxfp4", **other}
    name = next(iter(other))
    with pytest.raises(ValueError, match=name):
        MXFP4Config.from_config(config)
    with caplog.at_level(logging.WARNING):
        assert load_quantization_config(str(tmp_path), {"quantization_config": config}) is None
    assert name in caplog.text


def test_other_widths_are_no_config(tmp_path, caplog):
    with caplog.at_level(logging.WARNING):
        assert load_quantization_config(str(tmp_path), {"quantization_config": {"quant_method": "mxfp4", "bits": 8}}) is None
    assert "8 bits" in caplog.text


def test_keys_that_ask_for_nothing(tmp_path):
    for config in ({}, {"modules_to_not_convert": None}, {"modules_to_not_convert": [], "dequantize": False},
                   {"bits": 4, "group_size": 32, "is_checkpoint_mxfp4_serialized": False}):
        config = {"quant_method": "MXFP4", **config}
        assert isinstance(MXFP4Config.from_config(config), MXFP4Config)
        got = load_quantization_config(str(tmp_path), {"quantization_config": config})
        assert isinstance(got, MXFP4Config)
        assert got.is_checkpoint_mxfp4_serialized is config.get("is_checkpoint_mxfp4_serialized", True)


def test_capability():
    assert MXFP4Config().get_min_capability() == 95

"""The config keys of the operators around the step (no GPU)."""
import pytest

from patrickstar_b200.engine import parse_config


def test_both_are_off_by_default():
    for cfg in (None, {}, {"fp8": None}, {"fp8": {}}, {"fp8": {"enabled": False, "grad_format": "e5m2"}}):
        p = parse_config(cfg)
        assert p["fp8"] is None and p["distillation"] == {"temperature": 1.0, "tail": "drop", "weight": 1.0}


def test_values_and_refusals():
    assert parse_config({"fp8": {"enabled": True}})["fp8"] == "e4m3"
    assert parse_config({"fp8": {"enabled": True, "grad_format": "e5m2"}})["fp8"] == "e5m2"
    p = parse_config({"distillation": {"temperature": 2.0, "tail": "bucket"}})
    assert p["distillation"] == {"temperature": 2.0, "tail": "bucket", "weight": 1.0}
    assert parse_config(None)["distillation"]["temperature"] == 1.0    # the defaults are not what was set above
    for bad in ({"fp8": {"enabled": True, "grad_format": "e3m4"}}, {"fp8": {"enabled": True, "format": "e5m2"}}, {"distillation": {"tail": "rest"}},
                {"distillation": {"alpha": 0.5}}):
        with pytest.raises(ValueError):
            parse_config(bad)

"""What a model's configuration of its blocks is held to, on the CPU."""
import pytest

from train_gpt_b200.step import GPT, SMALL, StepConfig


def _cfg(**kw):
    return StepConfig(**{**SMALL, "mm": "bf16", "norm": "torch_reference", "loss": "torch", "optimizer": "torch", **kw})


@pytest.mark.parametrize("name", ["swiglue", "silu", "relu", "", "GELU"])
def test_an_unknown_activation_is_refused(name):
    with pytest.raises(ValueError, match="unknown activation"):
        GPT(_cfg(activation=name), "cpu")


@pytest.mark.parametrize("name", ["gelu", "relu2", "swiglu", "geglu", "reglu"])
def test_the_known_ones_are_not(name):
    assert GPT(_cfg(activation=name), "cpu").gated == name.endswith("glu")

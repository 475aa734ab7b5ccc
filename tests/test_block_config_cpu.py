"""What a model's configuration of its blocks is held to, on the CPU."""
import pytest
import torch

from train_gpt_b200 import fp8
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


@pytest.mark.parametrize("name", ["swiglu", "geglu", "reglu"])
@pytest.mark.parametrize("mlp,linears", [("unfused", 7), ("fused", 5)])
def test_unfused_gated_projections_go_by_mm(name, mlp, linears, monkeypatch):
    """As the plain feed-forward's do: each of a layer's seven matrices is one FP8 linear's."""
    seen = []

    def linear(a, w, **kw):
        seen.append(w)
        return a @ w
    monkeypatch.setattr(fp8, "block_scaled_matmul", linear)
    model = GPT(_cfg(activation=name, mm="fp8", mlp=mlp), "cpu")
    with torch.no_grad():
        model.raw_logits(torch.randint(0, SMALL["vocab_size"], (2, 16)))
    assert len(seen) == SMALL["n_layers"] * linears
    assert {id(w) for w in seen} == {id(w) for w in model.matrices()}

"""The model with a norm on both sides of a block, as far as it goes without a GPU: parameters, buckets, checkpoints, the plain form."""
import pytest
import torch

from train_gpt_b200 import checkpoint
from train_gpt_b200.step import GPT, SMALL, StepConfig


def _cfg(**kw):
    return StepConfig(**SMALL, mm="bf16", norm="torch_reference", loss="torch", optimizer="torch", activation="relu2", **kw)


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_model_trains_every_parameter(gate):
    model = GPT(_cfg(block_norm="sandwich", residual_gate=gate, residual_scale=0.9), "cpu")
    ids = torch.randint(0, 256, (2, 16))
    model.loss(ids, ids).backward()
    params = model.parameters()
    assert len({id(p) for p in params}) == len(params)
    assert all(p.grad is not None for p in params)
    plain = len(GPT(_cfg(), "cpu").parameters())
    assert len(params) == plain + 2 * SMALL["n_layers"] * (1 if gate == "none" else 2)


def test_the_junction_is_the_formula():
    cfg = _cfg(block_norm="sandwich", residual_gate="channel", residual_scale=0.5)
    model = GPT(cfg, "cpu")
    lp = model.layers[0]
    x, branch = torch.randn(2, 5, 128).to(torch.bfloat16), torch.randn(2, 5, 128).to(torch.bfloat16)
    x_new, h, _ = model._junction(x, branch, x, lp["norm2"], lp, 1)

    def rms(v):
        return v / torch.sqrt(v.square().mean(-1, keepdim=True) + cfg.rms_eps)
    want = 0.5 * x.double() + lp["gate1"].double() * rms(branch.double()) * lp["post1"].double()
    assert (x_new.double() - want).abs().max() <= 4 * 2.0 ** -8 * want.abs().max()
    assert (h.double() - rms(x_new.double())).abs().max() <= 4 * 2.0 ** -8 * h.double().abs().max()


def test_switches_that_need_each_other():
    for kw, message in ((dict(block_norm="post"), "block_norm"), (dict(block_norm="sandwich", residual_gate="head"), "residual_gate"),
                        (dict(residual_gate="channel"), "need block_norm"), (dict(residual_scale=0.5), "need block_norm")):
        with pytest.raises(ValueError, match=message):
            GPT(_cfg(**kw), "cpu")


def test_checkpoint_round_trip(tmp_path):
    a = GPT(_cfg(block_norm="sandwich", residual_gate="channel"), "cpu", seed=1)
    b = GPT(_cfg(block_norm="sandwich", residual_gate="channel"), "cpu", seed=2)
    with torch.no_grad():
        a.layers[1]["gate2"].mul_(3)
    tree, _, _ = checkpoint.load_checkpoint(checkpoint.save_checkpoint(tmp_path / "c.pkl", a, 3))
    checkpoint.load_params(b, tree)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    plain = GPT(_cfg(), "cpu")
    with pytest.raises(ValueError, match="layer parameters"):
        checkpoint.load_params(plain, tree)
    with pytest.raises(ValueError, match="layer parameters"):
        checkpoint.load_params(b, checkpoint.params_tree(plain))


def test_a_living_graph_is_seen():
    from train_gpt_b200.step import _graph_alive
    model = GPT(_cfg(), "cpu")
    ids = torch.randint(0, 256, (2, 16))
    assert not _graph_alive(model.parameters())
    loss = model.loss(ids, ids)
    assert _graph_alive(model.parameters())
    loss.backward()
    assert _graph_alive(model.parameters())
    del loss
    assert not _graph_alive(model.parameters()) and not _graph_alive(model.parameters())
    with torch.no_grad():
        kept = model.loss(ids, ids)
    assert not _graph_alive(model.parameters()) and kept.isfinite()

"""The model with rotary positions, normed queries and keys, a gated feed-forward and dropout, as far as it goes without a GPU: parameters, buckets,
checkpoints, the plain form."""
import numpy as np
import pytest
import torch

import block_reference as ref
from train_gpt_b200 import checkpoint
from train_gpt_b200.step import GPT, SMALL, StepConfig, Trainer, _keep, step_flops


def _cfg(**kw):
    kw = {"activation": "swiglu", "positions": "rotary", "qk_norm": True, **kw}
    return StepConfig(**SMALL, mm="bf16", norm="torch_reference", loss="torch", optimizer="torch", **kw)


@pytest.mark.parametrize("kw", [{}, dict(activation="geglu"), dict(activation="reglu", qk_norm=False), dict(activation="gelu"), dict(positions="learned"),
                                dict(dropout=0.3), dict(dropout=0.3, block_norm="sandwich")])
def test_model_trains_every_parameter(kw):
    cfg = _cfg(**kw)
    model = GPT(cfg, "cpu")
    ids = torch.randint(0, 256, (2, 16))
    loss = model.loss(ids, ids)
    loss.backward()
    params = model.parameters()
    assert torch.isfinite(loss) and len({id(p) for p in params}) == len(params) and all(p.grad is not None for p in params)
    plain = len(GPT(_cfg(activation="gelu", positions="learned", qk_norm=False), "cpu").parameters())
    more = (cfg.activation != "gelu") + 2 * cfg.qk_norm + 2 * (cfg.block_norm == "sandwich")
    assert len(params) == plain + SMALL["n_layers"] * more - (cfg.positions == "rotary")
    assert len(model.matrices()) == SMALL["n_layers"] * (6 if cfg.activation == "gelu" else 5)


def test_the_parts_are_the_formulas():
    cfg = _cfg(dropout=0.25)
    model = GPT(cfg, "cpu", seed=5)
    lp = model.layers[0]
    with torch.no_grad():
        lp["q_norm"].copy_(torch.rand(32) + 0.5)
    q, k = (torch.randn(2, 7, 4, 32).to(torch.bfloat16) for _ in range(2))
    at = torch.arange(7).expand(2, 7)
    for got, x, w in zip(model._place(q, k, lp), (q, k), (lp["q_norm"], lp["k_norm"])):
        want, size = ref.heads(x.double(), w.double(), at, cfg.rms_eps, cfg.rope_theta, 32, False)
        assert ((got.double() - want).abs() <= ref.BF * want.abs() + 2.0 ** -18 * size).all()
    h = torch.randn(2, 7, 128).to(torch.bfloat16)
    g, u = (h.double() @ lp[n].double() for n in ("w_gate", "w_up"))
    got, want = model._gated(h, lp).double(), ref.act(g, "silu")[0] * u
    # two projections and the activation rounded to bf16 before the product, and that: each 2^-8, through a slope of at most 1.13; the sums of 128 terms
    sums = [128 * ref.F32 * (h.double().abs() @ lp[n].double().abs()) for n in ("w_gate", "w_up")]
    most = 1.01 * (3 * ref.BF * want.abs() + 1.2 * (ref.BF * g.abs() + sums[0]) * u.abs() + 1.2 * sums[1] * g.abs())
    assert ((got - want).abs() <= most).all()
    y = model._drop(h, 3, h)
    mask, scale = ref.kept(h.numel(), 0.25, 5, 3)
    want = torch.where(torch.from_numpy(mask).view(h.shape), h.double() * scale, 0.0) + h.double()
    assert ((y.double() - want).abs() <= ref.BF * want.abs() + 2.0 ** -22 * (1 + scale) * h.double().abs()).all()


@pytest.mark.parametrize("n,seed,site", [(1, 0, 0), (8, -1, 7), (1003, 2 ** 62 + 12345, 2 ** 32 - 1), (4099, -2 ** 63, 3)])
def test_the_plain_mask_is_the_generators(n, seed, site):
    mask, _ = ref.kept(n, 0.4, seed, site)
    assert np.array_equal(_keep(torch.zeros(n), 0.4, torch.tensor([seed]), site).numpy(), mask)


def test_dropout_draws_anew_every_step_and_none_without_gradients():
    cfg = _cfg(dropout=0.5)
    tr = Trainer(cfg, "cpu", seed=3)
    ids = torch.randint(0, 256, (2, 16))
    with torch.no_grad():
        a, b = tr.model.loss(ids, ids), tr.model.loss(ids, ids)
    plain = GPT(_cfg(), "cpu", seed=3)
    with torch.no_grad():
        assert torch.equal(a, b) and torch.equal(a, plain.loss(ids, ids))
    first = tr.model.loss(ids, ids).detach()
    assert torch.equal(first, tr.model.loss(ids, ids).detach()) and not torch.equal(first, a)
    before = int(tr.model.dropout_seed)
    tr.step(ids, ids)
    assert int(tr.model.dropout_seed) == before + 1


def test_switches_that_are_refused():
    for kw, message in ((dict(positions="alibi"), "positions"), (dict(head_dim=24), "head_dim"), (dict(dropout=1.5), "dropout"), (dict(dropout=-0.1), "dropout")):
        with pytest.raises(ValueError, match=message):
            GPT(StepConfig(**{**SMALL, **{"mm": "bf16", "norm": "torch_reference", "positions": "rotary", **kw}}), "cpu")


def test_checkpoint_round_trip(tmp_path):
    a, b = GPT(_cfg(), "cpu", seed=1), GPT(_cfg(), "cpu", seed=2)
    with torch.no_grad():
        a.layers[1]["q_norm"].mul_(3)
    tree, _, _ = checkpoint.load_checkpoint(checkpoint.save_checkpoint(tmp_path / "c.pkl", a, 3))
    checkpoint.load_params(b, tree)
    assert "pos" not in tree and all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
    plain = GPT(_cfg(activation="gelu", positions="learned", qk_norm=False), "cpu")
    for model, other in ((plain, tree), (b, checkpoint.params_tree(plain))):
        with pytest.raises(ValueError, match="checkpoint has"):
            checkpoint.load_params(model, other)


def test_a_gated_layer_has_three_matrices_to_count():
    a, b = step_flops(_cfg(), 100), step_flops(_cfg(activation="gelu"), 100)
    assert a - b == 6.0 * SMALL["n_layers"] * SMALL["d_model"] * SMALL["d_ff"] * 100

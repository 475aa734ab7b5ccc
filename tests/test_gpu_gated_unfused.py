"""A model whose gated feed-forward's projections are linears of their own, by every `mm`: steps of it, launched one by one and captured."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{}, dict(activation="reglu"), dict(mm="fp8_ref"), dict(mm="bf16", norm="kernel"), dict(residual="separate"), dict(direct_grads=False)])
def test_every_parameter_gets_a_gradient(kw):
    from train_gpt_b200.step import SMALL, StepConfig, Trainer, synthetic_batch
    cfg = StepConfig(**{**SMALL, "vocab_size": 1001, "activation": "swiglu", "mlp": "unfused", **kw})
    runs = []
    for graph in (False, True):
        tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
        losses = []
        for i in range(3):
            loss, norm = tr.step(*synthetic_batch(cfg, 4, torch.device("cuda", 0), i))
            losses.append((float(loss), float(norm)))
            for bi in range(len(tr.buckets.flat)):
                for grad in tr.buckets.views(bi, tr.buckets.flat[bi]):
                    assert torch.isfinite(grad).all() and grad.any()
        runs.append((losses, [p.detach().clone() for p in tr.model.parameters()]))
        del tr
    assert runs[0][0] == runs[1][0] and all(torch.equal(p, q) for p, q in zip(runs[0][1], runs[1][1]))


def test_its_gradients_are_those_of_the_bf16_model_to_fp8s_roundings():
    import dataclasses
    from train_gpt_b200.step import GPT, SMALL, StepConfig, synthetic_batch
    cfg = StepConfig(**{**SMALL, "vocab_size": 1001, "activation": "swiglu", "mlp": "unfused"})
    ids, targets = synthetic_batch(cfg, 4, torch.device("cuda", 0), 1)
    a = GPT(cfg, torch.device("cuda", 0), seed=3)
    b = GPT(dataclasses.replace(cfg, mm="bf16", norm="kernel"), torch.device("cuda", 0), seed=3)
    for m in (a, b):
        m.loss(ids, targets).backward()
    for lp, lq in zip(a.layers, b.layers):
        for n in ("w_gate", "w_up", "w_down"):
            p, q = lp[n].grad.double(), lq[n].grad.double()
            # 2^-4 of each e4m3 operand: two of a product, in seven products of a layer one way and fourteen back, two layers: sqrt(84) of them in 2-norm
            assert float((p - q).norm()) <= 84 ** 0.5 * 2.0 ** -4 * float(q.norm())

"""A distillation step as it is used: a teacher's top logits, a student with a norm on both sides of its blocks, the loss against the
teacher, the optimiser's step, launched one by one and replayed as a graph."""
import dataclasses

import pytest
import torch

import operators_reference as ref

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    from train_gpt_b200.step import SMALL, StepConfig
    return StepConfig(**{**SMALL, "vocab_size": 1001}, activation="relu2", **kw)


def _batch(cfg, seed, batch=4):
    from train_gpt_b200.step import synthetic_batch
    return synthetic_batch(cfg, batch, torch.device("cuda", 0), seed)


def _teacher(cfg):
    from train_gpt_b200.step import GPT
    return GPT(dataclasses.replace(cfg, block_norm="pre", residual_gate="none", residual_scale=1.0), torch.device("cuda", 0), seed=99)


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_student_step(gate):
    """The loss is that of the student's own logits by the 64-bit form; every parameter gets a gradient."""
    from train_gpt_b200.step import Trainer
    cfg = _cfg(block_norm="sandwich", residual_gate=gate, residual_scale=0.9, distill_temperature=2.0, distill_weight=0.5)
    teacher = _teacher(cfg)
    ids, targets = _batch(cfg, 1)
    top = teacher.top_logits(ids, 32, cfg.distill_temperature)
    tr = Trainer(cfg, torch.device("cuda", 0), seed=3)
    assert tr._program is None
    with torch.no_grad():
        x = tr.model.raw_logits(ids).double().flatten(0, 1)
    want = ref.distill_rows(x, top.ids.flatten(0, 1), top.logp.flatten(0, 1), top.log_rest.flatten(), cfg.logit_cap, targets.flatten(), 2.0, 0.5).mean()
    loss, norm = tr.step(ids, targets, teacher=top)
    # the logits of two forward passes are the same bits; the loss is float32 of sums as tests of the loss bound them
    assert abs(float(loss) - float(want)) <= 1e-3 and float(norm) > 0
    # (a weight of 1 need not move: a step of 3e-4 is less than half of bf16's 2^-8 below 1)
    b = tr.buckets
    for bi in range(len(b.flat)):
        for grad in b.views(bi, b.flat[bi]):
            assert torch.isfinite(grad).all() and grad.any()


def test_junctions_gradients_reach_the_model():
    """The fused junction against the same model with torch's operators: the two differ by bf16 roundings inside the layers."""
    from train_gpt_b200.step import GPT
    cfg = _cfg(block_norm="sandwich", residual_gate="channel", residual_scale=0.9, mm="bf16", norm="kernel")
    a = GPT(cfg, torch.device("cuda", 0), seed=3)
    b = GPT(dataclasses.replace(cfg, norm="torch_reference"), torch.device("cuda", 0), seed=3)
    ids, targets = _batch(cfg, 1)
    for m in (a, b):
        m.loss(ids, targets).backward()
    for p, q in zip(a.parameters(), b.parameters()):
        p, q = p.grad.double(), q.grad.double()
        # a layer has six roundings of 2^-8 one way and as many back, two layers and the head: sqrt(30) of them in 2-norm, four times that allowed
        assert float((p - q).norm()) <= 4 * 30 ** 0.5 * 2.0 ** -8 * float(q.norm())


def test_graph_replays_the_eager_steps():
    """A captured step with a teacher follows the eager one, batch after batch, and refuses a teacher of another form."""
    from train_gpt_b200 import losses
    from train_gpt_b200.step import Trainer
    cfg = _cfg(block_norm="sandwich", residual_gate="channel", distill_temperature=2.0, distill_weight=0.5)
    teacher = _teacher(cfg)
    runs = []
    for graph in (False, True):
        tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
        seen = []
        for i in range(3):
            ids, targets = _batch(cfg, i)
            loss, norm = tr.step(ids, targets, teacher=teacher.top_logits(ids, 16, 2.0))
            seen.append((float(loss), float(norm)))
        runs.append(seen)
    # (attention's backward pass adds in no fixed order, which moves the parameters' last bits from the second step on)
    assert runs[0][0][0] == runs[1][0][0]
    for (a, b), (c, d) in zip(*runs):
        assert abs(a - c) <= 2e-3 * abs(a) and abs(b - d) <= 2e-2 * b
    ids, targets = _batch(cfg, 7)
    for bad in (None, teacher.top_logits(ids, 8, 2.0), teacher.top_logits(ids, 16, 2.0)._replace(log_rest=None)):
        with pytest.raises(ValueError, match="form that it was captured with"):
            tr.step(ids, targets, teacher=bad)
    assert isinstance(teacher.top_logits(ids, 8), losses.TopLogits)


def test_a_step_without_a_teacher_is_unchanged():
    """With the default switches the native program still runs, and a teacher only for one step leaves the next ones to it."""
    from train_gpt_b200.step import Trainer
    cfg = _cfg()
    tr, other = (Trainer(cfg, torch.device("cuda", 0), seed=3) for _ in range(2))
    assert tr._program is not None
    ids, targets = _batch(cfg, 1)
    a, b = tr.step(ids, targets), other.step(ids, targets)
    assert torch.equal(a[0], b[0])
    loss, _ = tr.step(ids, targets, teacher=_teacher(cfg).top_logits(ids, 16))
    assert torch.isfinite(loss)
    assert torch.isfinite(tr.step(ids, targets)[0])


def test_a_living_loss_refuses_the_capture():
    from train_gpt_b200.step import Trainer
    cfg = _cfg(distill_temperature=2.0, distill_weight=0.5)
    tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=True)
    ids, targets = _batch(cfg, 1)
    top = _teacher(cfg).top_logits(ids, 16, 2.0)
    loss = tr.model.distillation_loss(ids, targets, top)
    with pytest.raises(RuntimeError, match="still alive"):
        tr.step(ids, targets, teacher=top)
    want = loss.detach().clone()
    del loss
    got, _ = tr.step(ids, targets, teacher=top)
    assert torch.equal(got, want)

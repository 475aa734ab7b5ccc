"""A loss with dropout that is alive across a step: its masks were drawn from a seed that the step changes, whoever launches it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{}, dict(mm="bf16", norm="kernel")])
@pytest.mark.parametrize("graph", [False, True])
def test_a_loss_across_a_step_is_refused(graph, kw):
    from train_gpt_b200.step import SMALL, StepConfig, Trainer, synthetic_batch
    cfg = StepConfig(**{**SMALL, "vocab_size": 1001, "activation": "swiglu", "dropout": 0.2, **kw})
    tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
    batch = synthetic_batch(cfg, 4, torch.device("cuda", 0), 1)
    tr.step(*batch)
    loss = tr.model.loss(*batch)
    tr.step(*batch)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    del loss
    assert torch.isfinite(tr.step(*batch)[0])


def test_a_users_own_graph():
    from train_gpt_b200 import kernels
    x = torch.randn(64, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    seed = torch.tensor([5], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        seed.add_(1)
    y = kernels.dropout(x, 0.5, seed)
    graph.replay()
    torch.autograd.graph.increment_version(seed)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.float().sum().backward()

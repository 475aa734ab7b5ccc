"""The reference's FP8 linear (bf16 straight-through gradients) in captured graphs: a whole training step, and a call with its backward pass."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kw", [{}, dict(norm="kernel", activation="relu2", mlp="unfused")])
def test_a_captured_step_follows_the_eager_one(kw):
    from train_gpt_b200.step import SMALL, StepConfig, Trainer, synthetic_batch
    cfg = StepConfig(**{**SMALL, "mm": "fp8_ref", **kw})
    runs = []
    for graph in (False, True):
        tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
        seen = [[float(v) for v in tr.step(*synthetic_batch(cfg, 4, torch.device("cuda", 0), i))] for i in range(3)]
        runs.append((seen, [p.detach().clone() for p in tr.model.parameters()]))
        del tr
    assert runs[0][0] == runs[1][0] and all(torch.equal(p, q) for p, q in zip(runs[0][1], runs[1][1]))


def test_a_captured_call():
    from train_gpt_b200 import fp8
    gen = torch.Generator(device="cuda").manual_seed(0)
    a, b, g = (torch.randn(s, device="cuda", generator=gen).to(torch.bfloat16) for s in ((96, 256), (256, 384), (96, 384)))
    leaves = [a.requires_grad_(), b.requires_grad_()]

    def run():
        y = fp8.block_scaled_matmul(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(out, want))

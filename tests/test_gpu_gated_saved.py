"""What kernels.gated_linear saves for its backward pass is saved as torch's own operators save: hooks see it, checkpointing lets go of it."""
import pytest
import torch
from torch.utils.checkpoint import checkpoint

from train_gpt_b200 import kernels

pytestmark = pytest.mark.gpu


def _make(m, k, f):
    gen = torch.Generator(device="cuda").manual_seed(0)

    def rnd(*shape, std=1.0):
        return (std * torch.randn(shape, device="cuda", generator=gen)).to(torch.bfloat16)
    return [rnd(m, k).requires_grad_(), rnd(k, f, std=k ** -0.5).requires_grad_(), rnd(k, f, std=k ** -0.5).requires_grad_()], rnd(m, f)


def test_hooks_see_what_is_kept():
    leaves, g = _make(300, 64, 200)
    want = torch.autograd.grad(kernels.gated_linear(*leaves), leaves, g)
    seen = []

    def pack(t):
        seen.append((t.dtype, tuple(t.shape)))
        return t.cpu()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.cuda()):
        h = kernels.gated_linear(*leaves)
    assert seen.count((torch.float16, (300, 200))) == 2 and torch.uint8 in [d for d, _ in seen]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, leaves, g, retain_graph=True), want))
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, leaves, g), want))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(h, leaves, g)


def test_a_checkpointed_call_keeps_nothing():
    leaves, g = _make(4096, 64, 2048)
    want = torch.autograd.grad(kernels.gated_linear(*leaves), leaves, g)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    h = checkpoint(kernels.gated_linear, *leaves, use_reentrant=False)
    held = torch.cuda.memory_allocated() - before
    assert held < 1.5 * h.numel() * 2                # (the output; both projections would be twice as much again)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(h, leaves, g), want))

"""A teacher's answer made under torch.inference_mode(): its tensors count no changes, so that the loss cannot see that they were overwritten."""
import pytest
import torch

from test_gpu_distill import _logits, _teacher

pytestmark = pytest.mark.gpu


def _inference_teacher(vocab, targets):
    from train_gpt_b200 import losses
    teacher = losses.TopLogits(*_teacher(7, vocab, 8, 15.0, 1.0))
    with torch.inference_mode():
        made = losses.TopLogits(*(t.clone() for t in teacher))
        made_targets = targets.clone()
    assert all(t.is_inference() for t in (*made, made_targets))
    return teacher, made, made_targets


def test_it_is_taken_as_any_other():
    from train_gpt_b200 import losses
    targets = torch.randint(0, 300, (7,), device="cuda")
    plain, made, made_targets = _inference_teacher(300, targets)
    x = _logits(7, 300, seed=5)
    out = []
    for teacher, t in ((plain, targets), (made, made_targets)):
        leaf = x.clone().requires_grad_()
        loss = losses.capped_distillation(leaf, teacher, 15.0, target_ids=t, weight=0.5)
        loss.backward(torch.tensor(3.0, device="cuda"))
        out.append((loss.detach(), leaf.grad))
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
    with torch.inference_mode():
        x = _logits(7, 300, seed=5)
        top = losses.top_logits(x, 15.0, 8)
        loss = losses.capped_distillation(x, top, 15.0)
    assert top.ids.is_inference() and not loss.requires_grad


@pytest.mark.parametrize("which", ["ids", "logp", "log_rest", "targets"])
def test_overwritten_between_the_passes(which):
    """The next batch's answer may be written where this one's was while its loss waits for its backward pass."""
    from train_gpt_b200 import losses
    targets = torch.randint(0, 300, (7,), device="cuda")
    plain, made, made_targets = _inference_teacher(300, targets)
    x = _logits(7, 300, seed=5)
    leaf = x.clone().requires_grad_()
    (want,) = torch.autograd.grad(losses.capped_distillation(leaf, plain, 15.0, target_ids=targets, weight=0.5), leaf)
    loss = losses.capped_distillation(leaf, made, 15.0, target_ids=made_targets, weight=0.5)
    with torch.inference_mode():
        (made_targets if which == "targets" else getattr(made, which)).zero_()
    (got,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device="cuda"), retain_graph=True)
    assert torch.equal(got, 2 * want)                     # (a power of two: the same digits)
    (again,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device="cuda"))
    assert torch.equal(again, got)

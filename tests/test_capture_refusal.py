"""A step that goes through autograd is not captured while a loss of the same model is alive, whatever it is that takes it there."""
import pytest
import torch

from train_gpt_b200.step import SMALL, StepConfig, Trainer


def _trainer():
    return Trainer(StepConfig(**SMALL, mm="bf16", norm="torch_reference", loss="torch", optimizer="torch", activation="relu2"), "cpu")


class _Program:
    """Stands for the native program: whether it takes a step."""

    def __init__(self, takes):
        self.takes = takes

    def applies(self):
        return self.takes


class _Reached(Exception):
    pass


def _capture(tr, monkeypatch):
    """As far as the warm-up steps."""
    def reached(*a, **k):
        raise _Reached
    monkeypatch.setattr(torch.cuda, "Stream", reached)
    ids = torch.randint(0, 256, (2, 16))
    tr._capture(ids, ids)


@pytest.mark.parametrize("program", [None, _Program(False)], ids=["no program", "a program that declines"])
def test_a_living_loss_refuses_the_capture_of_any_step_through_autograd(program, monkeypatch):
    tr = _trainer()
    tr._program = program
    ids = torch.randint(0, 256, (2, 16))
    loss = tr.model.loss(ids, ids)
    with pytest.raises(RuntimeError, match="still alive"):
        _capture(tr, monkeypatch)
    del loss
    with pytest.raises(_Reached):
        _capture(tr, monkeypatch)


def test_a_step_of_the_native_program_is_captured_beside_a_living_loss(monkeypatch):
    tr = _trainer()
    tr._program = _Program(True)
    ids = torch.randint(0, 256, (2, 16))
    loss = tr.model.loss(ids, ids)
    with pytest.raises(_Reached):
        _capture(tr, monkeypatch)
    del loss


@pytest.mark.gpu
@pytest.mark.parametrize("through", ["switch", "frozen"])
def test_a_living_loss_on_the_gpu(through):
    """A configuration without a native program, and one whose program declines because a parameter is frozen: refused, and captured afterwards."""
    tr = Trainer(StepConfig(**SMALL, activation="relu2", **(dict(qkv="separate") if through == "switch" else {})), torch.device("cuda", 0), seed=3, graph=True)
    assert (tr._program is None) == (through == "switch")
    if through == "frozen":
        assert tr._program.applies()
        tr.model.pos.requires_grad_(False)
        assert not tr._program.applies()
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, SMALL["vocab_size"], (2, SMALL["seq_len"]), device="cuda", generator=g)
    loss = tr.model.loss(ids, ids)
    with pytest.raises(RuntimeError, match="still alive"):
        tr.step(ids, ids)
    want = loss.detach().clone()
    del loss
    got, _ = tr.step(ids, ids)
    assert torch.equal(got, want)

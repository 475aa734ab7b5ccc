"""Forward-mode derivatives of the distillation loss and of the sandwich norm are an error; both would be dropped otherwise."""
import pytest
import torch
from torch.autograd import forward_ad

BF = torch.bfloat16


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.fixture(params=["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def device(request):
    return request.param


@pytest.mark.parametrize("which", ["x", "branch", "post", "pre", "gate"])
def test_sandwich_norm(which, device):
    from train_gpt_b200 import kernels
    a = dict(x=torch.ones(4, 128, dtype=BF, device=device), branch=torch.ones(4, 128, dtype=BF, device=device), post=torch.ones(128, dtype=BF, device=device),
             pre=torch.ones(128, dtype=BF, device=device), gate=torch.ones(128, dtype=BF, device=device))
    with forward_ad.dual_level():
        a[which] = _dual(a[which])
        with pytest.raises(RuntimeError, match="sandwich_norm has no forward-mode derivative"):
            kernels.sandwich_norm(a["x"], a["branch"], a["post"], a["pre"], 1e-5, gate=a["gate"])


@pytest.mark.parametrize("which", ["logits", "logp", "log_rest"])
def test_capped_distillation(which, device):
    from train_gpt_b200 import losses
    a = dict(logits=torch.ones(2, 16, dtype=BF, device=device), logp=torch.zeros(2, 4, device=device), log_rest=torch.zeros(2, device=device))
    ids = torch.arange(4, dtype=torch.int32, device=device).expand(2, 4)
    with forward_ad.dual_level():
        a[which] = _dual(a[which])
        with pytest.raises(RuntimeError, match="capped_distillation has no forward-mode derivative"):
            losses.capped_distillation(a["logits"], losses.TopLogits(ids, a["logp"], a["log_rest"]), 15.0)


@pytest.mark.gpu
def test_a_level_without_a_tangent_changes_nothing():
    from train_gpt_b200 import kernels
    x, y, w = torch.ones(4, 128, dtype=BF, device="cuda"), torch.ones(4, 128, dtype=BF, device="cuda"), torch.ones(128, dtype=BF, device="cuda")
    want = kernels.sandwich_norm(x, y, w, w, 1e-5)
    with forward_ad.dual_level():
        got = kernels.sandwich_norm(x, y, w, w, 1e-5)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

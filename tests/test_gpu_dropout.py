"""kernels.dropout against Philox in NumPy: the same elements are dropped, the others within half a step of bf16 (2^-8) and two float32 roundings
(2^-22 of the terms) of residual + x / (1 - p)."""
import numpy as np
import pytest
import torch

from train_gpt_b200 import kernels

import block_reference as ref

pytestmark = pytest.mark.gpu


def _seed(v):
    return torch.tensor([v], device="cuda", dtype=torch.int64)


def _rnd(*shape, seed=0):
    return torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(torch.bfloat16)


def _want(x, p, seed, site, residual=None):
    mask, scale = ref.kept(x.numel(), p, seed, site)
    mask = torch.from_numpy(mask).to("cuda").view(x.shape)
    v = torch.where(mask, x.double() * scale, 0.0)
    return (v if residual is None else v + residual.double()), v.abs() + (0 if residual is None else residual.double().abs()), mask


def _check(x, p, seed, site=0, residual=None):
    want, size, mask = _want(x, p, seed, site, residual)
    got = kernels.dropout(x, p, _seed(seed), site, residual)
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    if residual is None:
        assert torch.equal(got != 0, mask & (x != 0))
    assert ((got.double() - want).abs() <= ref.BF * want.abs() + 2.0 ** -22 * size).all()
    return got


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 15, 16, 17, 255, 4096, 4099, 65543, 1000003])
@pytest.mark.parametrize("with_residual", [False, True])
def test_any_number_of_elements(n, with_residual):
    _check(_rnd(n, seed=n), 0.3, 12345 + n, 7, _rnd(n, seed=n + 1) if with_residual else None)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18, 2.0 ** -17, 1e-4, 0.05, 0.1, 0.5, 0.9, 65535 / 65536, 1 - 2.0 ** -17, 1 - 2.0 ** -18, 1.0])
def test_probabilities(p):
    x, r = _rnd(100003), _rnd(100003, seed=1)
    got = _check(x, p, 99, 3)
    _check(x, p, 99, 3, r)
    if p == 0.0:
        assert torch.equal(got, x)
    if p == 1.0:
        assert not got.any() and torch.equal(kernels.dropout(x, 1.0, _seed(1), residual=r), r)


@pytest.mark.parametrize("seed", [0, 1, -1, 2 ** 62, -2 ** 63, 2 ** 32, 0x123456789ABCDEF])
@pytest.mark.parametrize("site", [0, 1, 2 ** 32 - 1])
def test_seeds_and_sites(seed, site):
    _check(_rnd(8, 1003), 0.25, seed, site)


def test_masks_differ_and_keep_their_share():
    x = torch.ones(1 << 22, device="cuda", dtype=torch.bfloat16)
    masks = [kernels.dropout(x, 0.1, _seed(s), site) != 0 for s, site in ((1, 0), (1, 1), (2, 0))]
    n = x.numel()
    for i, m in enumerate(masks):                       # five standard deviations of n draws
        assert abs(float(m.sum()) - 0.9 * n) <= 5 * (0.09 * n) ** 0.5 + n * 2.0 ** -17
        for o in masks[:i]:
            assert abs(float((m & o).sum()) - 0.81 * n) <= 5 * (0.81 * 0.19 * n) ** 0.5 + n * 2.0 ** -16


@pytest.mark.parametrize("with_residual", [False, True])
def test_gradients(with_residual):
    x, r, g = _rnd(5, 1031).requires_grad_(), _rnd(5, 1031, seed=1).requires_grad_(), _rnd(5, 1031, seed=2)
    y = kernels.dropout(x, 0.4, _seed(5), 2, r if with_residual else None)
    y.backward(g)
    want, size, _ = _want(g, 0.4, 5, 2)
    assert ((x.grad.double() - want).abs() <= ref.BF * want.abs() + 2.0 ** -22 * size).all()
    if with_residual:
        assert torch.equal(r.grad, g)
    (a, b), s = (x.detach().double(), r.detach().double()), 1e-3
    step = torch.randn(x.shape, device="cuda", dtype=torch.float64)
    mask, scale = ref.kept(x.numel(), 0.4, 5, 2)
    mask = torch.from_numpy(mask).to("cuda").view(x.shape)
    f = lambda v: ((torch.where(mask, v * scale, 0.0) + b) * g.double()).sum()                      # noqa: E731
    assert abs((f(a + s * step) - f(a - s * step)) / (2 * s) - (x.grad.double() * step).sum()) <= 2 * ref.BF * (x.grad.double() * step).abs().sum()


def test_dropped_elements_are_zero_whatever_they_are():
    x = torch.full((4096,), float("nan"), device="cuda", dtype=torch.bfloat16)
    x[::2] = float("inf")
    mask, _ = ref.kept(4096, 0.5, 3, 0)
    mask = torch.from_numpy(mask).to("cuda")
    y = kernels.dropout(x, 0.5, _seed(3))
    assert not y[~mask].any() and torch.equal(y[mask].isnan(), x[mask].isnan()) and y[mask][~x[mask].isnan()].isinf().all()
    r = torch.ones_like(x)
    assert (kernels.dropout(x, 0.5, _seed(3), residual=r)[~mask] == 1).all()


def test_strides_alignment_and_places():
    x = _rnd(64, 72)
    want = kernels.dropout(x, 0.2, _seed(4))
    wide = torch.zeros(64, 80, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:75] = x
    assert torch.equal(kernels.dropout(wide[:, 3:75], 0.2, _seed(4)), want)
    assert torch.equal(kernels.dropout(x.T.contiguous().T, 0.2, _seed(4)), want)
    assert torch.equal(kernels.dropout(x.view(8, 8, 72), 0.2, _seed(4)).view(64, 72), want)
    r = _rnd(64, 72, seed=9)
    assert torch.equal(kernels.dropout(x, 0.2, _seed(4), residual=wide[:, 3:75]), kernels.dropout(x, 0.2, _seed(4), residual=x))
    seeds = torch.tensor([1, 4], device="cuda")
    assert torch.equal(kernels.dropout(x, 0.2, seeds[1:]), want) and torch.equal(kernels.dropout(x, 0.2, seeds[1]), want)
    assert kernels.dropout(x[:0], 0.2, _seed(4)).shape == (0, 72)
    assert r.shape == x.shape


def test_in_place_through_the_c_entry():
    from train_gpt_b200 import _lib
    lib, x, r, s = _lib.load(), _rnd(1009), _rnd(1009, seed=1), _seed(8)
    want = kernels.dropout(x, 0.3, s, 1, r)
    st = torch.cuda.current_stream().cuda_stream
    for y in (x.clone(), r.clone()):
        a, b = (y, r) if torch.equal(y, x) else (x, y)
        assert lib.tg_dropout(a.data_ptr(), b.data_ptr(), 0.3, s.data_ptr(), 1, y.data_ptr(), 1009, st) == 0
        assert torch.equal(y, want)


def test_a_graph_draws_what_the_seed_says():
    x, s = _rnd(300, 100).requires_grad_(), _seed(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(kernels.dropout(x, 0.5, s, 3).sum(), x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = kernels.dropout(x, 0.5, s, 3)
        dx, = torch.autograd.grad(y, x, torch.ones_like(y))
        y = y.detach()
        s.add_(1)
    for seed in (1, 2, 3):
        graph.replay()
        want = kernels.dropout(x.detach(), 0.5, _seed(seed), 3)
        assert torch.equal(y, want) and torch.equal(dx != 0, want != 0)


def test_the_seed_may_not_change_before_the_backward_pass():
    x, s = _rnd(64).requires_grad_(), _seed(1)
    y = kernels.dropout(x, 0.5, s)
    s.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(RuntimeError, match="differentiable once"):
        g = torch.ones(64, device="cuda", dtype=torch.bfloat16).requires_grad_()
        d, = torch.autograd.grad(kernels.dropout(x, 0.5, s), x, g, create_graph=True)
        d.sum().backward()


def test_far_elements():
    """A mask beyond 2^32 elements of a tensor's start."""
    n = 2 ** 32 + 2 ** 12 + 5
    x = torch.empty(n, device="cuda", dtype=torch.bfloat16)
    x[-8192:] = 1
    y = kernels.dropout(x, 0.5, _seed(6))
    first = n - 8192
    mask, _ = ref.kept(8192, 0.5, 6, 0, first)
    assert np.array_equal((y[-8192:] != 0).cpu().numpy(), mask)

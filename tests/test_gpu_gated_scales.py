"""kernels.gated_linear's gradients where the projections are small, or of very different sizes: what the forward pass keeps of them is right relative to
the largest of 64 columns, at any scale."""
import pytest
import torch

from train_gpt_b200 import kernels, ops

import block_reference as ref

pytestmark = pytest.mark.gpu

# few tokens, in two pieces; the contraction in ranges; tiles on pairs of SMs, ragged
SIZES = [(40, 64, 200), (24, 2048, 72), (1100, 64, 2504)]


def _make(m, k, f):
    def rnd(*shape, std=1.0, seed=0):
        return (std * torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).to(torch.bfloat16)
    return rnd(m, k, seed=1), rnd(k, f, std=k ** -0.5, seed=2), rnd(k, f, std=k ** -0.5, seed=3), rnd(m, f, seed=4)


def _kept(v, acc, smallest):
    """How far a projection v, accumulated to acc, may be off when the backward pass sees it: half a step of fp16, and `smallest` of the largest finite one of
    its 64 columns, which is scaled into [2^14, 2^15) where the smallest steps are 2^-24."""
    top = torch.where(torch.isfinite(v), v.abs() + acc, 0.0)
    top = torch.stack([p.amax(1) for p in top.split(64, 1)], 1).repeat_interleave(64, 1)[:, :v.shape[1]]
    return acc + ref.F16 * v.abs() + smallest * top


def _want(x, wg, wu, act, grad):
    """[(value, how far it may be off), ...] of dx, dw_gate, dw_up; a relu's slope goes by the sign that was accumulated, whatever is kept"""
    k, (m, f) = x.shape[1], grad.shape
    g, u = x @ wg, x @ wu
    acc_g, acc_u = (k * ref.F32 * (x.abs() @ w.abs()) for w in (wg, wu))
    eg, eu = _kept(g, acc_g, 2.0 ** (-38 if act == "relu" else -39)), _kept(u, acc_u, 2.0 ** -39)
    a, da = ref.act(g, act)
    bend = (g.abs() <= acc_g).double() if act == "relu" else (0.8 * eg).clamp_max(1.2) + (2.0 ** -20 * (1 + g.abs())).clamp_max(1.2)
    dg, du = grad * u * da, grad * a
    err_g = ref.BF * dg.abs() + grad.abs() * (bend * (u.abs() + eu) + 1.2 * eu)
    err_u = ref.BF * du.abs() + grad.abs() * (1.2 * eg + 2.0 ** -20 * g.abs())

    def total(value, parts, n):
        return value, 1.01 * ref.BF * value.abs() + sum(1.01 * (p.abs() @ e) + 2 * n * ref.F32 * (p.abs() @ q.abs()) for p, q, e in parts) + 1e-38
    dx = (dg @ wg.T + du @ wu.T).T
    dx, e = total(dx, [(wg, dg.T, err_g.T), (wu, du.T, err_u.T)], 2 * f)
    return [(dx.T, e.T), total(x.T @ dg, [(x.T, dg, err_g)], m), total(x.T @ du, [(x.T, du, err_u)], m)]


def _grads(x, wg, wu, act, g):
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(kernels.gated_linear(*leaves, act), leaves, g)
    ops.check_status()
    return grads


def _check(x, wg, wu, act, g, columns=slice(None)):
    for got, (value, most), name in zip(_grads(x, wg, wu, act, g), _want(*[t.double() for t in (x, wg, wu)], act, g.double()), ("dx", "dw_gate", "dw_up")):
        if name != "dx":
            got, value, most = got[:, columns], value[:, columns], most[:, columns]
        elif columns != slice(None):
            continue
        off = (got.double() - value).abs()
        assert torch.isfinite(got).all() and (off <= most).all(), (name, float((off / most).max()))
        assert float(most.norm()) <= 0.5 * float(value.norm())        # (the bound says something)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("power", [-20, -40, -60])
@pytest.mark.parametrize("what", ["x", "weights", "w_gate", "w_up"])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_small_projections(m, k, f, what, power, act):
    x, wg, wu, g = _make(m, k, f)
    s = 2.0 ** power
    if what == "x":
        x = x * s
    if what in ("weights", "w_gate"):
        wg = wg * s
    if what in ("weights", "w_up"):
        wu = wu * s
    if what in ("x", "weights"):
        g = g / s                                # (products of two small ones stay within bf16's range)
    _check(x, wg, wu, act, g)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_a_large_projection_beside_ordinary_ones(m, k, f, act):
    """One column of 64 2^16 times the others: those have eleven bits all the same."""
    x, wg, wu, g = _make(m, k, f)
    wg, wu, g = wg.clone(), wu.clone(), g.clone()
    wg[:, 7] *= 2.0 ** 16
    wu[:, 66] *= 2.0 ** 16
    g[:, 7] *= 2.0 ** -16
    g[:, 66] *= 2.0 ** -16
    _check(x, wg, wu, act, g)


def test_zeros():
    """Rows of which nothing is kept: no scale makes them anything else."""
    for m, k, f in SIZES:
        x, wg, wu, g = _make(m, k, f)
        x[1] = 0
        for act in ("silu", "gelu", "relu"):
            dx, _, _ = _grads(x, wg, wu, act, g)
            _, dg, du = _grads(torch.zeros_like(x), wg, wu, act, g)
            assert not dx[1].any() and not dg.any() and not du.any()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("m,k,f", SIZES)
def test_what_is_not_finite_stays_in_its_column(m, k, f, value, act):
    x, wg, wu, g = _make(m, k, f)
    wg, wu = wg.clone(), wu.clone()
    wg[3, 7] = wu[5, 9] = wu[1, 66] = value
    columns = torch.ones(f, dtype=torch.bool, device="cuda")
    columns[[7, 9, 66]] = False
    _check(x, wg, wu, act, g, columns)
    dx, dg, du = _grads(x, wg, wu, act, g)
    assert not torch.isfinite(dg[:, 9]).any() and not torch.isfinite(dg[:, 66]).any()


@pytest.mark.parametrize("m,k,f", SIZES)
def test_a_positive_gate_keeps_its_slope(m, k, f):
    """relu: beside one that is 2^45 times as large, too."""
    x, wg, wu, g = _make(m, k, f)
    wg = wg.clone()
    wg[:, ::64] *= 2.0 ** 45
    _, (want, most), _ = _want(*[t.double() for t in (x, wg, wu)], "relu", g.double())
    _, got, _ = _grads(x, wg, wu, "relu", g)
    assert ((got.double() - want).abs() <= most).all() and float(most.norm()) <= 0.5 * float(want.norm())

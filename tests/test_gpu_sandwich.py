"""kernels.sandwich_norm and its backward pass against their 64-bit forms.

Tolerances.  A result is rounded to bf16 once: 2^-8 of it.  Before that everything is float32: a factor (a square root of a mean, its
reciprocal) is off by a few 2^-24 of itself, each product and sum by 2^-24 of its size; 2^-20 of the summands' sizes holds sixteen of them.
A sum over the rows has at most one rounding per row and block, so (rows + 256) 2^-24 of its summands' sizes beside that."""
import pytest
import torch

import operators_reference as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5
BF = 2.0 ** -8


def _inputs(shape, gate, seed=0, dev="cuda"):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(s, scale=1.0):
        return (scale * torch.randn(s, device=dev, generator=g)).to(torch.bfloat16)

    d = shape[-1]
    x, y = normal(shape, 2.0), normal(shape)
    y.view(-1)[:: 97] *= 30                                            # outlier features
    post, pre = (1 + 0.1 * torch.randn(2, d, device=dev, generator=g)).to(torch.bfloat16)
    gate = {"none": None, "channel": normal((d,)), "token": normal((*shape[:-1], 1))}[gate]
    return x, y, post, pre, gate, normal(shape), normal(shape)


def _near(got, want, size, extra=2.0 ** -20):
    got = got.double()
    bad = (got - want).abs() > BF * want.abs() + extra * size
    assert not bad.any(), (int(bad.sum()), float(((got - want).abs() / (BF * want.abs() + extra * size)).max()))


def _f(t):
    return None if t is None else t.detach().double()


def _check(x, y, post, pre, gate, alpha, g, gh, quantize=False):
    from train_gpt_b200 import kernels, ops
    leaves = [t.detach().clone().requires_grad_() for t in (x, y, post, pre) + (() if gate is None else (gate,))]
    gate_l = leaves[4] if gate is not None else None
    out = kernels.sandwich_norm(*leaves[:4], EPS, gate=gate_l, residual_scale=alpha, quantize=quantize)
    x_new, h = out[:2]
    d = x.shape[-1]
    x2, y2, g2, gh2, n2 = (_f(t).reshape(-1, d) for t in (x, y, g, gh, x_new))
    gate2 = None if gate is None else _f(gate) if gate.shape == (d,) and gate.dim() == 1 else _f(gate).reshape(-1, 1)
    want, size = ref.sandwich(x2, y2, _f(post), _f(pre), EPS, gate2, alpha)
    _near(x_new.detach().reshape(-1, d), want, size)
    want_h = ref.rms(n2, EPS) * _f(pre)                                # the norm of x' as it is kept
    _near(h.detach().reshape(-1, d), want_h, want_h.abs())
    if quantize:
        q, s = ops.quantize_rowwise(h.detach())
        assert torch.equal(out[2].view(torch.uint8), q.view(torch.uint8)) and torch.equal(out[3], s)
        assert not out[2].requires_grad and not out[3].requires_grad
    grads = torch.autograd.grad((x_new, h), leaves, (g, gh))
    wants = ref.sandwich_bwd(n2, y2, _f(post), _f(pre), EPS, gate2, alpha, g2, gh2)
    rows = x2.shape[0]
    for name, got in zip(("dx", "dbranch", "dpost", "dpre", "dgate"), grads):
        value, size = wants[name]
        over_rows = got.dim() == 1 and name not in ("dx", "dbranch") and not (name == "dgate" and gate.dim() > 1)
        _near(got.reshape(value.shape), value, size, 2.0 ** -20 + ((rows + 256) * 2.0 ** -24 if over_rows else 0.0))
    return x_new, h, grads


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 128), (129, 256), (33, 264), (700, 1024), (50, 1032), (1000, 2048), (7, 1536), (65, 2304), (300, 4096), (5, 5000),
                                       (40, 6144), (16, 8192), (600, 8184), (5000, 520), (2500, 768), (1600, 1288), (1300, 2824), (500, 2560), (700, 3464), (333, 4616), (300, 7000)])
def test_against_the_formulas(rows, cols, gate):
    _check(*_inputs((rows, cols), gate)[:5], 0.9, *_inputs((rows, cols), gate)[5:])


@pytest.mark.parametrize("rows,cols", [(1, 128), (200, 384), (1000, 1024), (257, 2048), (16, 8192), (31, 4224), (2500, 768), (1600, 1280), (1300, 2944), (700, 5120)])
def test_quantised_form(rows, cols):
    i = _inputs((rows, cols), "channel", seed=3)
    _check(*i[:5], 1.0, *i[5:], quantize=True)


def test_quantised_inference_form():
    from train_gpt_b200 import kernels, ops
    x, y, post, pre, gate, _, _ = _inputs((4, 9, 512), "token")
    x_new, h = kernels.sandwich_norm_quant(x, y, post, pre, EPS, gate=gate, residual_scale=0.5, want_y=True)
    a, b = kernels.sandwich_norm(x, y, post, pre, EPS, gate=gate, residual_scale=0.5)
    assert torch.equal(x_new, a) and torch.equal(h.y, b)
    q, s = ops.quantize_rowwise(b)
    assert torch.equal(h.q.view(torch.uint8), q.view(torch.uint8)) and torch.equal(h.scales, s)
    assert kernels.sandwich_norm_quant(x, y, post, pre, EPS, gate=gate, residual_scale=0.5)[1].y is None


def test_leading_shape_strides_and_alignment():
    """A batch of sequences; a branch that is a slice of a wider matrix, vectors that begin 2 bytes past a boundary."""
    x, y, post, pre, gate, g, gh = _inputs((3, 17, 384), "token", seed=1)
    wide = torch.zeros(3, 17, 400, dtype=torch.bfloat16, device="cuda")
    wide[..., 5:389] = y
    shifted = torch.empty(385, dtype=torch.bfloat16, device="cuda")
    shifted[1:] = post
    want = _check(x, y, post, pre, gate, 1.0, g, gh)
    from train_gpt_b200 import kernels
    x_new, h = kernels.sandwich_norm(x, wide[..., 5:389], shifted[1:], pre, EPS, gate=gate)
    assert torch.equal(x_new, want[0]) and torch.equal(h, want[1])
    t = x.transpose(0, 1).contiguous().transpose(0, 1)                  # same values, other strides
    assert torch.equal(kernels.sandwich_norm(t, y, post, pre, EPS, gate=gate)[0], want[0])


def test_one_gradient_missing():
    """Only h, or only x', is used: the other's gradient is zero."""
    from train_gpt_b200 import kernels
    x, y, post, pre, gate, g, gh = _inputs((90, 640), "channel", seed=2)
    for use in (0, 1):
        leaves = [t.clone().requires_grad_() for t in (x, y, post, pre, gate)]
        out = kernels.sandwich_norm(*leaves[:4], EPS, gate=leaves[4])
        only = torch.autograd.grad(out[use], leaves, (g, gh)[use])
        leaves2 = [t.clone().requires_grad_() for t in (x, y, post, pre, gate)]
        out2 = kernels.sandwich_norm(*leaves2[:4], EPS, gate=leaves2[4])
        zeros = torch.zeros_like(g)
        both = torch.autograd.grad(out2, leaves2, (g, zeros) if use == 0 else (zeros, gh))
        for a, b in zip(only, both):
            assert torch.equal(a, b)


def test_against_differences():
    """Along random directions: the change of sum(g x' + gh h) by the 64-bit form, against the gradients' inner product; the rounding of
    x' is left out of the 64-bit form, which moves h by 2^-8 of itself."""
    x, y, post, pre, gate, g, gh = _inputs((20, 256), "channel", seed=5)
    _, _, grads = _check(x, y, post, pre, gate, 0.9, g, gh)
    gen = torch.Generator(device="cuda").manual_seed(1)

    def value(x, y, post, pre, gate):
        n, _ = ref.sandwich(x, y, post, pre, EPS, gate, 0.9)
        return (g.double() * n).sum() + (gh.double() * (ref.rms(n, EPS) * pre)).sum()

    at = [_f(t) for t in (x, y, post, pre, gate)]
    for i, grad in enumerate(grads):
        v = torch.randn(at[i].shape, device="cuda", generator=gen, dtype=torch.float64)
        step = 1e-5
        plus, minus = ([a + (s * step * v if j == i else 0.0) for j, a in enumerate(at)] for s in (1, -1))
        diff = (value(*plus) - value(*minus)) / (2 * step)
        size = (grad.double() * v).abs().sum()
        assert abs(float(diff - (grad.double() * v).sum())) <= 3 * BF * float(size)


def test_rows_of_zeros_and_large_values():
    """A branch of zeros has a factor of 1 / sqrt(eps) and stays zero; values near the type's largest do not overflow the sums of squares
    (float32 reaches 3.4e38: rows of 256 values of 1e18 are 2.6e38)."""
    from train_gpt_b200 import kernels
    x, y, post, pre, gate, g, gh = _inputs((6, 256), "channel", seed=6)
    y[1] = 0
    x[2] = 0
    y[2] = 0
    x[3] = 1e18
    y[4] = 1e18
    _check(x, y, post, pre, gate, 1.0, g, gh)


def test_nan_stays_in_its_row():
    from train_gpt_b200 import kernels
    x, y, post, pre, gate, _, _ = _inputs((12, 512), "none", seed=7)
    clean = kernels.sandwich_norm(x, y, post, pre, EPS)
    y[5, 3] = float("nan")
    x[9, 7] = float("inf")
    x_new, h = kernels.sandwich_norm(x, y, post, pre, EPS)
    assert x_new[5].isnan().all() and h[5].isnan().all() and x_new[9, 7].isinf() and h[9, 7].isnan()
    keep = [i for i in range(12) if i not in (5, 9)]
    assert torch.equal(x_new[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep])


def test_no_rows():
    from train_gpt_b200 import kernels
    leaves = [t.requires_grad_() for t in (torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda"),
                                           torch.ones(64, dtype=torch.bfloat16, device="cuda"), torch.ones(64, dtype=torch.bfloat16, device="cuda"),
                                           torch.ones(64, dtype=torch.bfloat16, device="cuda"))]
    x_new, h = kernels.sandwich_norm(*leaves[:4], EPS, gate=leaves[4])
    assert x_new.shape == h.shape == (0, 64)
    grads = torch.autograd.grad((x_new, h), leaves, (torch.zeros_like(x_new), torch.zeros_like(h)))
    assert all(not t.any() for t in grads[2:])


def test_in_place_changes_and_second_derivatives_are_errors():
    from train_gpt_b200 import kernels
    x, y, post, pre, _, g, gh = _inputs((4, 64), "none")
    y.requires_grad_()
    x_new, h = kernels.sandwich_norm(x, y, post, pre, EPS)
    with torch.no_grad():
        x_new.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.backward(gh)
    x_new, h = kernels.sandwich_norm(x, y, post, pre, EPS)
    gg = gh.clone().requires_grad_()
    (dy,) = torch.autograd.grad(h, y, gg, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        dy.sum().backward()
    x_new, h = kernels.sandwich_norm(x, y, post, pre, EPS)
    h.backward(gh)
    with pytest.raises(RuntimeError, match="second time"):
        h.backward(gh)


def test_same_bits_on_other_streams_and_in_a_graph():
    from train_gpt_b200 import ops
    x, y, post, pre, gate, g, gh = _inputs((333, 1024), "token", seed=8)

    def call():
        x_new, h, _, _ = ops.sandwich_norm_fwd(x, y, post, pre, EPS, gate=gate, residual_scale=0.7)
        return [x_new, h, *ops.sandwich_norm_bwd(x_new, y, post, pre, EPS, g, gh, gate=gate, residual_scale=0.7)]

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    with torch.no_grad():
        y.mul_(0.5)
    want = call()
    for graph, out in graphs:
        graph.replay()
    for graph, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))

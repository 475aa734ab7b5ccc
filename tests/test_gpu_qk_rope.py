"""kernels.qk_norm_rope and its backward pass against their 64-bit forms.

Tolerances.  An output is rounded to bf16 once: 2^-8 of the value.  Before that, float32: a norm's sum of up to 512 squares in a tree, its root and
three products are within 2^-19; a sine within 2^-22 of the angle's, the angle within 2^-22 (2^-18 for positions up to 2^31).  Together 2^-18 (2^-17) of the
magnitudes that a value is made of; the backward pass has twice the steps.  A scale's gradient is a sum of n terms, in float32 and any
order: n 2^-24 of the terms' magnitudes more."""
import pytest
import torch

from train_gpt_b200 import kernels, ops

import block_reference as ref

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _near(got, want, size, steps, what):
    off = (got.double() - want).abs()
    most = ref.BF * want.abs() + steps * size
    assert torch.isfinite(got).all(), what
    assert (off <= most).all(), (what, float((off / most.clamp_min(1e-300)).max()))


def _make(lead, heads, kv, dim, seed=0, scales=True, packed=False):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*shape):
        return torch.randn(shape, device="cuda", generator=g).to(torch.bfloat16)
    if packed:
        x = rnd(*lead, (heads + 2 * kv) * dim)
        q, k = x[..., :heads * dim].unflatten(-1, (heads, dim)), x[..., heads * dim:(heads + kv) * dim].unflatten(-1, (kv, dim))
    else:
        q, k = rnd(*lead, heads, dim), rnd(*lead, kv, dim)
    w = [(1 + 0.3 * torch.randn(dim, device="cuda", generator=g)).to(torch.bfloat16) if scales else None for _ in range(2)]
    return q, k, w[0], w[1], rnd(*lead, heads, dim), rnd(*lead, kv, dim)


def _check(q, k, wq, wk, gq, gk, positions=None, theta=10000.0, rotary=None, interleaved=False, steps=2.0 ** -18):
    dim = q.shape[-1]
    rotary = dim if rotary is None else rotary
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (q, k, wq, wk)]
    out = kernels.qk_norm_rope(*leaves, EPS, positions, theta=theta, rotary_dim=rotary, interleaved=interleaved)
    lead = q.shape[:-2]
    at = torch.arange(lead[-1], device="cuda").expand(lead) if positions is None and lead else positions if positions is not None else torch.zeros((), device="cuda")
    at = at.expand(lead)
    ins = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(out, ins, (gq, gk))
    for i, (x, w, g, name) in enumerate(((q, wq, gq, "q"), (k, wk, gk, "k"))):
        xd, wd = x.double(), None if w is None else w.double()
        want, size = ref.heads(xd, wd, at, EPS, theta, rotary, interleaved)
        assert out[i].is_contiguous() and out[i].shape == x.shape
        _near(out[i], want, size, steps, name)
        dx, dsize, dw, wsize = ref.heads_bwd(xd, wd, g.double(), at, EPS, theta, rotary, interleaved)
        _near(grads[i], dx, dsize, 2 * steps, "d" + name)
        if w is not None:
            n = x.numel() // dim
            _near(grads[2 + i], dw, wsize, 2 * steps + n * 2.0 ** -24, f"d{name}_scale")
    with torch.no_grad():
        again = kernels.qk_norm_rope(*leaves, EPS, positions, theta=theta, rotary_dim=rotary, interleaved=interleaved)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])
    return out, grads


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 256, 272, 384, 512])
@pytest.mark.parametrize("interleaved", [False, True])
def test_every_kind_of_head(dim, interleaved):
    _check(*_make((2, 5), 3, 2, dim, seed=dim), interleaved=interleaved)


@pytest.mark.parametrize("dim,rotary", [(64, 0), (64, 16), (64, 48), (80, 32), (96, 80), (128, 16), (256, 240), (512, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("scales", [False, True])
def test_a_part_of_the_head(dim, rotary, interleaved, scales):
    q, k, wq, wk, gq, gk = _make((3, 7), 4, 1, dim, seed=rotary, scales=scales)
    out, _ = _check(q, k, wq, wk, gq, gk, rotary=rotary, interleaved=interleaved)
    if not scales:
        assert torch.equal(out[0][..., rotary:], q[..., rotary:])


@pytest.mark.parametrize("lead,heads,kv", [((1, 1), 1, 1), ((1, 1), 64, 8), ((16, 1), 32, 8), ((1,), 5, 3), ((), 7, 2), ((2, 3, 4), 3, 3), ((1, 2049), 2, 1), ((301, 1), 9, 3),
                                           ((1, 3), 1, 40), ((5, 700), 16, 16)])
def test_shapes(lead, heads, kv):
    _check(*_make(lead, heads, kv, 64, seed=heads))


@pytest.mark.parametrize("scales", [False, True])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("shape", [(3, 6), (6,), (3, 1), (1,), ()])
def test_positions(scales, dtype, shape):
    g = torch.Generator(device="cuda").manual_seed(len(shape))
    positions = torch.randint(-1000, 200000, shape, device="cuda", generator=g).to(dtype)
    _check(*_make((3, 6), 4, 2, 128, seed=3, scales=scales), positions=positions, theta=500000.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions_far_away(interleaved):
    positions = torch.tensor([[2 ** 31 - 1, 2 ** 24 + 1, 10 ** 6], [-(2 ** 31) + 1, 0, 10 ** 9]], device="cuda")
    _check(*_make((2, 3), 4, 2, 64), positions=positions, theta=1e6, interleaved=interleaved, steps=2.0 ** -17)


def test_positions_with_strides():
    wide = torch.randint(0, 5000, (6, 8), device="cuda")
    _check(*_make((3, 6), 2, 2, 64), positions=wide[:, ::2].T[:3, :], theta=300.0)


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_slices_of_one_projection_are_read_as_they_lie(dim):
    args = _make((2, 19), 6, 2, dim, packed=True)
    assert not args[0].is_contiguous()
    out, grads = _check(*args)
    same, again = _check(args[0].contiguous(), args[1].contiguous(), *args[2:])
    assert all(torch.equal(a, b) for a, b in zip([*out, *grads], [*same, *again]))


def test_other_strides_are_read_or_copied():
    q, k, wq, wk, gq, gk = _make((2, 9), 4, 4, 64)
    want, dwant = _check(q, k, wq, wk, gq, gk)
    t = q.transpose(1, 2).contiguous().transpose(1, 2)                          # (batch, heads, tokens, dim)
    u = torch.empty((2, 9, 4, 64, 2), device="cuda", dtype=torch.bfloat16)
    u[..., 1] = k                                                              # no unit stride
    shifted = torch.empty(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view_as(q).copy_(q)       # two bytes off
    for a, b, x, y in ((t, u[..., 1], gq.transpose(1, 2).contiguous().transpose(1, 2), gk), (shifted, k, gq, gk.permute(3, 1, 0, 2).contiguous().permute(2, 1, 3, 0))):
        got, dgot = _check(a, b, wq, wk, x, y)
        assert all(torch.equal(v, w) for v, w in zip([*got, *dgot], [*want, *dwant]))
    one = torch.randn(1, 9, 1, 64, device="cuda").to(torch.bfloat16)
    _check(one.expand(2, 9, 4, 64), k, wq, wk, gq, gk)
    w = torch.empty(129, device="cuda", dtype=torch.bfloat16)
    w[1:65] = wq
    assert torch.equal(kernels.qk_norm_rope(q, k, w[1:65], wk, EPS)[0], want[0])


def test_no_tokens():
    for lead in ((0, 5), (3, 0), (0,)):
        args = _make(lead, 2, 1, 64)
        out, grads = _check(*args)
        assert all(not g.any() for g in grads[2:])


def test_extreme_heads():
    """Zeros, the largest values and not-a-number: each head on its own."""
    q, k, wq, wk, gq, gk = _make((1, 4), 3, 1, 64)
    clean = kernels.qk_norm_rope(q, k, wq, wk, EPS)
    d = kernels.qk_norm_rope
    bad = q.clone()
    bad[0, 1, 1] = 0
    bad[0, 2, 0, 5] = float("nan")
    bad[0, 3, 2, 7] = float("inf")
    out = d(bad, k, wq, wk, EPS)
    assert not out[0][0, 1, 1].any()
    assert out[0][0, 2, 0].isnan().all()
    hit = torch.zeros(1, 4, 3, dtype=torch.bool, device="cuda")
    for at in ((1, 1), (2, 0), (3, 2)):
        hit[0, at[0], at[1]] = True
    assert torch.equal(out[0][~hit], clean[0][~hit]) and torch.equal(out[1], clean[1])
    small = q * 2.0 ** -100
    want, size = ref.heads(small.double(), wq.double(), torch.arange(4, device="cuda").expand(1, 4), EPS, 10000.0, 64, False)
    _near(d(small, k, wq, wk, EPS)[0], want, size, 2.0 ** -18, "small")


def test_one_output_used():
    q, k, wq, wk, gq, gk = _make((2, 5), 3, 2, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    dq, dk, dwq, dwk = torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS)[0], leaves, gq)
    both = torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS), leaves, (gq, torch.zeros_like(gk)))
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dwq, dwk), both)) and not dk.any() and not dwk.any() and dwq.any()


def test_differences():
    """The gradient against differences of the 64-bit form: one that makes the same mistake as the formula would not agree with it."""
    q, k, wq, wk, gq, gk = _make((2, 4), 2, 1, 32)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS), leaves, (gq, gk))
    at = torch.arange(4, device="cuda").expand(2, 4)

    def loss(x, w, g):
        return (ref.heads(x, w, at, EPS, 10000.0, 32, False)[0] * g.double()).sum()
    gen = torch.Generator(device="cuda").manual_seed(1)
    for x, w, g, dx, dw in ((q, wq, gq, grads[0], grads[2]), (k, wk, gk, grads[1], grads[3])):
        for which, d in ((0, dx), (1, dw)):
            v = [x.double(), w.double()]
            step = torch.randn(v[which].shape, device="cuda", dtype=torch.float64, generator=gen)
            ends = []
            for s in (1, -1):
                u = list(v)
                u[which] = v[which] + s * 1e-5 * step
                ends.append(loss(*u, g))
            slope, got = (ends[0] - ends[1]) / 2e-5, (d.double() * step).sum()
            assert abs(slope - got) <= 2 * ref.BF * (d.double() * step).abs().sum(), which


def test_a_side_stream_and_a_graph():
    q, k, wq, wk, gq, gk = _make((2, 33), 4, 2, 64)
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    positions = torch.arange(33, device="cuda")

    def run():
        out = ops.qk_norm_rope_fwd(q, k, wq, wk, EPS, positions)
        return [*out, *ops.qk_norm_rope_bwd(q, k, gq, gk, wq, wk, EPS, positions)]
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    q.copy_(torch.randn(q.shape, device="cuda"))
    positions.add_(1000)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, run()))
    out = kernels.qk_norm_rope(*leaves, EPS, positions)
    graph2 = torch.cuda.CUDAGraph()
    del out
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS, positions), leaves, (gq, gk))
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph2):
        grads = torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS, positions), leaves, (gq, gk))
    gq.mul_(2)
    graph2.replay()
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS, positions), leaves, (gq, gk))))


def test_once_and_not_again():
    leaves = [t.detach().requires_grad_() for t in _make((1, 3), 2, 1, 32)[:4]]
    out = kernels.qk_norm_rope(*leaves, EPS)
    out[0].sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        out[0].sum().backward()
    d, = torch.autograd.grad(kernels.qk_norm_rope(*leaves, EPS)[0].float().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()
    x = leaves[0].detach().clone().requires_grad_()
    y = x * 1
    out = kernels.qk_norm_rope(y, *leaves[1:], EPS)
    y.data.mul_(1)
    with torch.no_grad():
        y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out[0].sum().backward()

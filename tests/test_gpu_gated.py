"""kernels.gated_linear and its backward pass against their 64-bit forms, within the bounds that block_reference makes from the roundings on
the way: float32 accumulation, fp16 of what is kept, bf16 of the gradients at the projections and of the results."""
import pytest
import torch

from train_gpt_b200 import kernels, ops

import block_reference as ref

pytestmark = pytest.mark.gpu


def _rnd(*shape, std=1.0, seed=0):
    return (std * torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).to(torch.bfloat16)


def _make(m, k, f, std=1.0):
    return _rnd(m, k, std=std, seed=1), _rnd(k, f, std=k ** -0.5, seed=2), _rnd(k, f, std=k ** -0.5, seed=3), _rnd(m, f, seed=4)


def _near(got, want, what):
    value, most = want
    assert got.shape == value.shape and torch.isfinite(got).all(), what
    off = (got.double() - value).abs()
    assert (off <= most).all(), (what, float((off / most).max()))


def _check(x, wg, wu, g, act="silu"):
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = kernels.gated_linear(*leaves, act)
    d = [t.double() for t in (x, wg, wu, g)]
    _near(h, ref.gated(*d[:3], act), "h")
    grads = torch.autograd.grad(h, leaves, g)
    for got, want, name in zip(grads, ref.gated_bwd(*d[:3], act, d[3]), ("dx", "dw_gate", "dw_up")):
        _near(got, want, name)
    with torch.no_grad():                       # (the same kernel, without what a backward pass needs)
        _near(kernels.gated_linear(*leaves, act), ref.gated(*d[:3], act), "h alone")
    ops.check_status()
    return h, grads


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("m,k,f", [(1, 8, 8), (3, 64, 64), (128, 128, 128), (130, 136, 200), (257, 72, 264), (300, 520, 1000), (1, 1024, 512), (700, 64, 24)])
def test_sizes(act, m, k, f):
    _check(*_make(m, k, f), act)


@pytest.mark.parametrize("m", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256])
def test_few_tokens(m):
    _check(*_make(m, 264, 392))


@pytest.mark.parametrize("k", [8, 16, 56, 64, 72, 120, 128, 136, 192, 512, 1000])
def test_contractions(k):
    _check(*_make(40, k, 136))


@pytest.mark.parametrize("f", [8, 56, 64, 72, 120, 128, 136, 248, 256, 264, 504, 512, 520])
def test_widths(f):
    _check(*_make(300, 96, f))


def test_many_tiles():
    _check(*_make(2309, 320, 2056))


def test_long_contractions():
    _check(*_make(24, 8192, 64))
    _check(*_make(9000, 16, 40))


@pytest.mark.parametrize("m,k,f", [(9000, 200, 72), (30000, 64, 520), (40, 1000, 8192), (130, 24, 16384), (20000, 2048, 40), (260, 264, 6000)])
def test_contractions_in_ranges(m, k, f):
    """Few tiles of a long contraction, of dx, of the weights' gradients or of both."""
    from train_gpt_b200 import _lib
    x, wg, wu, g = _make(m, k, f)
    _, grads = _check(x, wg, wu, g)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = kernels.gated_linear(*leaves)
    for which in ((0,), (1, 2), (0, 1, 2)):
        again = torch.autograd.grad(h, [leaves[i] for i in which], g, retain_graph=True)
        d = [t.double() for t in (x, wg, wu, g)]
        for got, want in zip(again, [ref.gated_bwd(*d[:3], "silu", d[3])[i] for i in which]):
            _near(got, want, which)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))
    lib = _lib.load()
    args = _lib.GatedArgs(x=16, ldx=k, w_gate=16, ld_gate=f, w_up=16, ld_up=f, dx=16, dw_gate=16, dw_up=16, rows=m, cols=k, inner=f)
    import ctypes
    assert lib.tg_gated_linear_bwd_scratch_bytes(ctypes.byref(args)) > 2 * ((m * f * 2 + 255) // 256 * 256)      # (it is cut)


def test_leading_axes_strides_and_alignment():
    x, wg, wu, g = _make(60, 64, 72)
    h, (dx, dg, du) = _check(x, wg, wu, g)
    shaped = [t.detach().requires_grad_() for t in (x.view(3, 4, 5, 64), wg, wu)]
    h2 = kernels.gated_linear(*shaped)
    assert h2.shape == (3, 4, 5, 72) and torch.equal(h2.view(60, 72), h)
    d2 = torch.autograd.grad(h2, shaped, g.view(3, 4, 5, 72))
    assert torch.equal(d2[0], dx.view(3, 4, 5, 64)) and torch.equal(d2[1], dg) and torch.equal(d2[2], du)
    both = torch.cat((wg, wu), 1)                                                # the weights side by side in one matrix
    wide = torch.zeros(60, 80, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:72] = x
    shifted = torch.zeros(60 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(60, 64).copy_(x)
    for a, b, c, gr in ((wide[:, 8:72], both[:, :72], both[:, 72:], g), (shifted, wg.T.contiguous().T, wu, g.T.contiguous().T),
                        (x, wg, wu, torch.cat((g, g), 1)[:, 72:])):
        again = [t.detach().requires_grad_() for t in (a, b, c)]
        h3 = kernels.gated_linear(*again)
        assert torch.equal(h3, h)
        assert all(torch.equal(p, q) for p, q in zip(torch.autograd.grad(h3, again, gr), (dx, dg, du)))
    with torch.no_grad():
        want = kernels.gated_linear(x, wg, wu)
        for a, b, c in ((wide[:, 8:72], both[:, :72], both[:, 72:]), (shifted, wg.T.contiguous().T, wu)):
            assert torch.equal(kernels.gated_linear(a, b, c), want)
    one = kernels.gated_linear(x[3], wg, wu)                                      # a token without a leading axis
    assert one.shape == (72,) and torch.equal(one, kernels.gated_linear(x[3:4], wg, wu)[0])
    row = x[:1].expand(60, 64)
    assert torch.equal(kernels.gated_linear(row, wg, wu)[7:8], kernels.gated_linear(row, wg, wu)[:1])


def test_no_rows():
    x, wg, wu, g = _make(0, 64, 72)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = kernels.gated_linear(*leaves)
    grads = torch.autograd.grad(h, leaves, g)
    assert h.shape == (0, 72) and grads[0].shape == (0, 64) and not grads[1].any() and not grads[2].any()


@pytest.mark.parametrize("which", [(0,), (1,), (2,), (0, 1), (1, 2)])
def test_some_gradients(which):
    x, wg, wu, g = _make(50, 72, 80)
    _, want = _check(x, wg, wu, g)
    leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((x, wg, wu))]
    got = torch.autograd.grad(kernels.gated_linear(*leaves), [leaves[i] for i in which], g)
    assert all(torch.equal(a, want[i]) for a, i in zip(got, which))


def test_one_weight_twice():
    x, w, _, g = _make(40, 64, 64)
    leaf = w.detach().requires_grad_()
    got, = torch.autograd.grad(kernels.gated_linear(x, leaf, leaf), leaf, g)
    _, (_, dg, du) = _check(x, w, w, g)
    assert torch.equal(got, dg + du)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
def test_projections_beyond_fp16(act):
    """What is kept has bf16's range: a power of two per 64 columns of a row."""
    x, wg, wu, g = _make(70, 64, 200)
    x = x.clone()
    x[3] *= 2.0 ** 20
    x[5] *= 2.0 ** -20
    x[6] *= 2.0 ** 50
    wu = wu.clone()
    wu[:, 70] *= 2.0 ** 30
    scale = torch.ones(70, 1, device="cuda", dtype=torch.bfloat16)
    scale[3], scale[6] = 2.0 ** -40, 2.0 ** -100
    g = g * scale
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = kernels.gated_linear(*leaves, act)
    dx, dg, du = torch.autograd.grad(h, leaves, g)
    assert torch.isfinite(dx).all() and torch.isfinite(dg).all() and torch.isfinite(du).all()
    # Each row of dx on its own: a row's projections are kept with its own exponents.  Values far below the largest of their 64 columns may be
    # off by its 2^-25, which the bound of the whole row covers with the largest projection in place of each one.
    xd, gd, ud, grad = (t.double() for t in (x, wg, wu, g))
    G, U = xd @ gd, xd @ ud
    a, da = ref.act(G, act)
    want = (grad * U * da) @ gd.T + (grad * a) @ ud.T
    top_g, top_u = G.abs().amax(1, keepdim=True), U.abs().amax(1, keepdim=True)
    eg, eu = (64 * ref.F32 * (xd.abs() @ w.abs()) + ref.F16 * v.abs() + 2.0 ** -24 * (1 + t) for w, v, t in ((gd, G, top_g), (ud, U, top_u)))
    bend = (G.abs() <= eg).double() if act == "relu" else torch.minimum(0.8 * eg, torch.full_like(eg, 1.2)) + 2.0 ** -20 * (1 + G.abs()).clamp_max(2.0 ** 20)
    off = (ref.BF * (grad * U * da).abs() + grad.abs() * (bend * (U.abs() + eu) + 1.2 * eu)) @ gd.abs().T + (ref.BF * (grad * a).abs() + grad.abs() * (1.2 * eg + 2.0 ** -20 * G.abs())) @ ud.abs().T
    off = 1.01 * (off + ref.BF * want.abs()) + 400 * ref.F32 * ((grad * U * da).abs() @ gd.abs().T + (grad * a).abs() @ ud.abs().T)
    assert ((dx.double() - want).abs() <= off).all()


@pytest.mark.parametrize("m", [1, 5, 64, 65, 128, 129, 300, 700])
@pytest.mark.parametrize("k,f", [(64, 64), (512, 64), (1000, 8), (1024, 512), (2048, 1096), (264, 18960), (72, 40000)])
def test_few_tokens_alone(m, k, f):
    """Without a gradient: one to eight ranges of the contraction, tiles beyond one round of the SMs."""
    x, wg, wu, _ = _make(m, k, f)
    d = [t.double() for t in (x, wg, wu)]
    for act in ("silu", "gelu", "relu"):
        with torch.no_grad():
            h = kernels.gated_linear(x, wg, wu, act)
            _near(h, ref.gated(*d, act), act)
            assert torch.equal(kernels.gated_linear(x, wg, wu, act), h)
    ops.check_status()


def test_few_tokens_in_graphs():
    x, wg, wu, _ = _make(7, 512, 264)
    with torch.no_grad():
        graphs = []
        kernels.gated_linear(x, wg, wu)
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs = [kernels.gated_linear(x, wg, wu, a) for a in ("silu", "gelu", "relu") * 3]
            graphs.append((g, outs))
        x.mul_(0.5)
        want = [kernels.gated_linear(x, wg, wu, a) for a in ("silu", "gelu", "relu") * 3]
        for g, outs in graphs:
            g.replay()
        assert all(torch.equal(a, b) for _, outs in graphs for a, b in zip(outs, want))
    ops.check_status()


@pytest.mark.parametrize("m,k,f", [(16, 1024, 1024), (300, 1024, 1024), (700, 512, 704)])
def test_two_streams_and_two_graphs_at_once(m, k, f):
    """A column tile's rows in one and in several blocks, the contraction in ranges: nothing is shared between calls."""
    x, wg, wu, _ = _make(m, k, f)
    xs = [x, x.flip(0).contiguous()]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    with torch.no_grad():
        want = [kernels.gated_linear(v, wg, wu) for v in xs]
        for v in xs:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                outs.append(kernels.gated_linear(v, wg, wu))
        for h in outs:
            h.fill_(float("nan"))
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for _ in range(20):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        alone = []
        for s, v in zip(streams, xs):
            with torch.cuda.stream(s):
                alone.append([kernels.gated_linear(v, wg, wu) for _ in range(5)])
        torch.cuda.synchronize()
    assert all(torch.equal(h, w) for h, w in zip(outs, want)) and all(torch.equal(h, w) for hs, w in zip(alone, want) for h in hs)
    ops.check_status()


@pytest.mark.parametrize("m", [5, 100, 300])
def test_rows_that_share_memory(m):
    """Expanded and overlapping rows, a column slice with a step."""
    x, wg, wu, _ = _make(m, 64, 128)
    wide = _make(m, 128, 128)[0]
    long = _make(m + 8, 64, 8)[0].flatten()
    for a, b in ((x[:1].expand(m, 64), wg), (long.as_strided((m, 64), (8, 1)), wg), (wide[:, ::2], wg), (x, wg[:1].expand(64, 128)), (x, wg.t().contiguous().t())):
        with torch.no_grad():
            assert torch.equal(kernels.gated_linear(a, b, wu), kernels.gated_linear(a.contiguous(), b.contiguous(), wu))


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("m,k,f", [(1, 8, 8), (56, 64, 64), (34, 80, 136), (65, 72, 72), (128, 128, 512), (130, 1000, 264), (2, 6488, 136), (500, 40, 1048)])
def test_small_problems_have_the_gradients_in_two_pieces(act, m, k, f):
    x, wg, wu, g = _make(m, k, f)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    grads = torch.autograd.grad(kernels.gated_linear(*leaves, act), leaves, g)
    for got, want, name in zip(grads, ref.gated_bwd(*[t.double() for t in (x, wg, wu)], act, g.double(), 2), ("dx", "dw_gate", "dw_up")):
        _near(got, want, name)


def test_an_infinite_gradient_stays_one():
    """Its second piece is zero, not the not-a-number that is left of it."""
    x, wg, wu, g = _make(40, 64, 72)
    g[3, 5] = float("inf")
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    dx, dg, du = torch.autograd.grad(kernels.gated_linear(*leaves), leaves, g)
    want = x[3].double() * torch.nn.functional.silu(x[3].double() @ wg.double())[5]
    assert torch.equal(du[:, 5].isposinf(), want > 0) and torch.equal(du[:, 5].isneginf(), want < 0)
    rest = torch.ones(72, dtype=torch.bool, device="cuda")
    rest[5] = False
    assert torch.isfinite(du[:, rest]).all() and torch.isfinite(dg[:, rest]).all()
    rows = torch.ones(40, dtype=torch.bool, device="cuda")
    rows[3] = False
    assert torch.isfinite(dx[rows]).all() and not torch.isfinite(dx[3]).any()


@pytest.mark.parametrize("m,k,f", [(40, 64, 72), (300, 64, 264), (24, 4096, 64)])
def test_the_least_scratch_does(m, k, f):
    """The C entry with room for one piece alone."""
    from train_gpt_b200 import _lib
    import ctypes
    lib, (x, wg, wu, g) = _lib.load(), _make(m, k, f)
    half = (m * f * 2 + 255) // 256 * 256
    h, kept = torch.empty_like(g), torch.empty(2, m, f, device="cuda", dtype=torch.float16)
    exponents = torch.empty(lib.tg_gated_linear_exponent_bytes(m, f), device="cuda", dtype=torch.uint8)
    out = [torch.empty_like(t) for t in (x, wg, wu)]
    scratch = torch.full((2 * half + 256,), 0x7F, device="cuda", dtype=torch.uint8)
    args = _lib.GatedArgs(x=x.data_ptr(), ldx=k, w_gate=wg.data_ptr(), ld_gate=f, w_up=wu.data_ptr(), ld_up=f, act=_lib.TG_GATED["silu"], h=h.data_ptr(),
                          saved_gate=kept[0].data_ptr(), saved_up=kept[1].data_ptr(), saved_exponents=exponents.data_ptr(), g=g.data_ptr(), dx=out[0].data_ptr(),
                          dw_gate=out[1].data_ptr(), dw_up=out[2].data_ptr(), scratch=scratch.data_ptr(), scratch_bytes=2 * half, rows=m, cols=k, inner=f)
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.tg_gated_linear_fwd(ctypes.byref(args), stream) == 0 and lib.tg_gated_linear_bwd(ctypes.byref(args), stream) == 0
    torch.cuda.synchronize()
    for got, want, name in zip(out, ref.gated_bwd(*[t.double() for t in (x, wg, wu)], "silu", g.double()), ("dx", "dw_gate", "dw_up")):
        _near(got, want, name)
    assert (scratch[2 * half:] == 0x7F).all()


def test_large_negative_gates_and_infinities():
    """silu and gelu go to 0 on the left, not to not-a-number; what is not finite stays in its row."""
    x, wg, wu, g = _make(40, 64, 64)
    wg = torch.eye(64, device="cuda", dtype=torch.bfloat16)
    clean = [kernels.gated_linear(x, wg, wu, a) for a in ("silu", "gelu", "relu")]
    big = x.clone()
    big[2] = -3000.0
    big[4, 3] = float("nan")
    big[6, 5] = float("inf")
    rest = torch.ones(40, dtype=torch.bool, device="cuda")
    rest[[2, 4, 6]] = False
    for a, want in zip(("silu", "gelu", "relu"), clean):
        h = kernels.gated_linear(big, wg, wu, a)
        assert not h[2].any() and torch.equal(h[rest], want[rest]) and h[4].isnan().any() and (~torch.isfinite(h[6])).any()


def test_differences():
    x, wg, wu, g = _make(20, 32, 40)
    for act in ("silu", "gelu"):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        grads = torch.autograd.grad(kernels.gated_linear(*leaves, act), leaves, g)
        v = [t.double() for t in (x, wg, wu)]
        gen = torch.Generator(device="cuda").manual_seed(7)
        for i, d in enumerate(grads):
            step = torch.randn(v[i].shape, device="cuda", dtype=torch.float64, generator=gen)
            ends = []
            for s in (1, -1):
                u = list(v)
                u[i] = v[i] + s * 1e-5 * step
                ends.append((ref.gated(*u, act)[0] * g.double()).sum())
            # (bf16 of the result, and of the gradients at the projections, whose share is as large)
            assert abs((ends[0] - ends[1]) / 2e-5 - (d.double() * step).sum()) <= 4 * ref.BF * (d.double() * step).abs().sum(), (act, i)


def test_a_side_stream_two_graphs_and_twice_at_once():
    x, wg, wu, g = _make(300, 128, 264)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]

    def run():
        h = kernels.gated_linear(*leaves)
        return [h.detach(), *torch.autograd.grad(h, leaves, g)]
    want = run()
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in sides:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append([run() for _ in range(4)])
    for s in sides:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for runs in got for r in runs for a, b in zip(r, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run()
        graphs.append((graph, out))
    with torch.no_grad():
        leaves[0].mul_(0.5)
    fresh = run()
    for graph, out in graphs:
        graph.replay()
    assert all(torch.equal(a, b) for _, out in graphs for a, b in zip(out, fresh))
    ops.check_status()


def test_once_and_not_again():
    x, wg, wu, g = _make(20, 32, 40)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
    h = kernels.gated_linear(*leaves)
    first = torch.autograd.grad(h, leaves, g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(h, leaves, g)))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(h, leaves, g)
    d, = torch.autograd.grad(kernels.gated_linear(*leaves).float().sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.sum().backward()

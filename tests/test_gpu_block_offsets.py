"""Heads and rows that lie beyond 2^31 elements and 2^32 bytes of their tensor's start: the same bits as those alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _room(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GB")


def _rnd(*shape, std=1.0, seed=0):
    return (std * torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))).to(torch.bfloat16)


@pytest.mark.parametrize("scales", [False, True])
def test_heads(scales):
    """2 x 300000 tokens of 48 + 16 heads of 64: the queries alone are 1.8 10^9 elements, with the keys and values behind them in one projection 3.1 10^9."""
    from train_gpt_b200 import ops
    _room(60)
    B, T, H, K, D, few = 2, 300000, 48, 16, 64, 37
    tail = _rnd(few, (H + 2 * K) * D, seed=1)
    big = torch.zeros(B, T, (H + 2 * K) * D, dtype=torch.bfloat16, device="cuda")
    big[-1, -few:] = tail

    def heads(t):
        return t[..., :H * D].unflatten(-1, (H, D)), t[..., H * D:(H + K) * D].unflatten(-1, (K, D))
    w = [1 + _rnd(D, std=0.1, seed=s) for s in (2, 3)] if scales else [None, None]
    at = torch.arange(T, device="cuda")
    q, k = heads(big)
    qt, kt = heads(tail[None])
    out, want = ops.qk_norm_rope_fwd(q, k, *w, EPS, at), ops.qk_norm_rope_fwd(qt, kt, *w, EPS, at[-few:])
    assert all(torch.equal(a[-1, -few:], b[0]) for a, b in zip(out, want)) and not out[0][0].any()
    gt = (_rnd(1, few, H, D, seed=4), _rnd(1, few, K, D, seed=5))
    g = (out[0].zero_(), out[1].zero_())
    for a, b in zip(g, gt):
        a[-1, -few:] = b[0]
    d, dwant = ops.qk_norm_rope_bwd(q, k, *g, *w, EPS, at), ops.qk_norm_rope_bwd(qt, kt, *gt, *w, EPS, at[-few:])
    assert all(torch.equal(a[-1, -few:], b[0]) for a, b in zip(d[:2], dwant[:2])) and not d[0][0].any()
    if scales:      # the same terms, and zeros, added up in another order: 37 tokens of 48 heads, and bf16 of the sum
        for a, b in zip(d[2:], dwant[2:]):
            assert float((a.double() - b.double()).abs().max()) <= 2 * 2.0 ** -8 * float(b.double().abs().max())


def test_rows():
    """150000 x 16 -> 16384: h, what is kept and the gradients at the projections have 2.5 10^9 elements each."""
    from train_gpt_b200 import kernels, ops
    _room(60)
    m, k, f, few = 150000, 16, 16384, 300
    xt, wg, wu, gt = _rnd(few, k, seed=1), _rnd(k, f, std=0.25, seed=2), _rnd(k, f, std=0.25, seed=3), _rnd(few, f, seed=4)
    x, g = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda"), torch.zeros(m, f, dtype=torch.bfloat16, device="cuda")
    x[-few:], g[-few:] = xt, gt
    leaves, alone = [t.detach().requires_grad_() for t in (x, wg, wu)], [t.detach().requires_grad_() for t in (xt, wg, wu)]
    h, want = kernels.gated_linear(*leaves), kernels.gated_linear(*alone)
    assert torch.equal(h[-few:], want) and not h[:-few].any()
    grads, dwant = torch.autograd.grad(h, leaves, g), torch.autograd.grad(want, alone, gt)
    # (the same sums in ranges that may be cut elsewhere: float32 of 2 x 16384 and of 300 terms, a rounding to bf16 behind each)
    for a, b in zip((grads[0][-few:], *grads[1:]), dwant):
        a, b = a.double(), b.double()
        assert ((a - b).abs() <= 2 * 2.0 ** -8 * b.abs() + 2.0 ** -12 * b.square().mean().sqrt()).all()
    assert not grads[0][:-few].any()
    with torch.no_grad():
        assert torch.equal(kernels.gated_linear(x, wg, wu)[-few:], want)
    ops.check_status()

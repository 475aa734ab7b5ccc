"""A block's operators together, as a model uses them: queries and keys normed and rotated out of one projection, attention, dropout with the
residual add, a gated feed-forward; a training step, launched one by one and replayed as a graph."""
import dataclasses

import pytest
import torch

pytestmark = pytest.mark.gpu


def _cfg(**kw):
    from train_gpt_b200.step import SMALL, StepConfig
    return StepConfig(**{**SMALL, "vocab_size": 1001, **{"activation": "swiglu", "positions": "rotary", "qk_norm": True, "dropout": 0.2, **kw}})


def _batch(cfg, seed, batch=4):
    from train_gpt_b200.step import synthetic_batch
    return synthetic_batch(cfg, batch, torch.device("cuda", 0), seed)


@pytest.mark.parametrize("kw", [{}, dict(activation="geglu"), dict(activation="reglu", qk_norm=False), dict(block_norm="sandwich"), dict(positions="learned")])
def test_the_model_with_the_kernels_and_without(kw):
    """The same model with torch's operators in place of the block's, its masks drawn the same: the two differ by bf16 roundings inside the layers."""
    from train_gpt_b200.step import GPT
    cfg = _cfg(mm="bf16", norm="kernel", **kw)
    a = GPT(cfg, torch.device("cuda", 0), seed=3)
    b = GPT(dataclasses.replace(cfg, norm="torch_reference"), torch.device("cuda", 0), seed=3)
    ids, targets = _batch(cfg, 1)
    for m in (a, b):
        m.loss(ids, targets).backward()
    for p, q in zip(a.parameters(), b.parameters()):
        p, q = p.grad.double(), q.grad.double()
        # a layer has ten roundings of 2^-8 one way and as many back, two layers and the head: sqrt(44) of them in 2-norm, four times that allowed
        assert float((p - q).norm()) <= 4 * 44 ** 0.5 * 2.0 ** -8 * float(q.norm())


@pytest.mark.parametrize("kw", [{}, dict(mm="fp8_ref"), dict(mm="bf16", norm="kernel"), dict(block_norm="sandwich", residual_gate="channel"), dict(dropout=0.0),
                                dict(qkv="separate", residual="separate"), dict(activation="gelu"), dict(positions="learned", qk_norm=False)])
def test_every_parameter_gets_a_gradient(kw):
    from train_gpt_b200.step import Trainer
    cfg = _cfg(**kw)
    tr = Trainer(cfg, torch.device("cuda", 0), seed=3)
    assert tr._program is None
    for i in range(2):
        loss, norm = tr.step(*_batch(cfg, i))
        assert torch.isfinite(loss) and float(norm) > 0
        for bi in range(len(tr.buckets.flat)):
            for grad in tr.buckets.views(bi, tr.buckets.flat[bi]):
                assert torch.isfinite(grad).all() and grad.any()


@pytest.mark.parametrize("kw", [{}, dict(mm="bf16", norm="kernel")])
def test_graph_replays_the_eager_steps(kw):
    """A captured step follows the eager one, batch after batch, masks included."""
    from train_gpt_b200.step import Trainer
    cfg = _cfg(**kw)
    runs = []
    for graph in (False, True):
        tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
        seen = []
        for i in range(4):
            loss, norm = tr.step(*_batch(cfg, i))
            seen.append((float(loss), float(norm)))
        runs.append((seen, int(tr.model.dropout_seed), [p.detach().clone() for p in tr.model.parameters()]))
        del tr
    assert runs[0][0] == runs[1][0] and runs[0][1] == runs[1][1]
    assert all(torch.equal(p, q) for p, q in zip(runs[0][2], runs[1][2]))


def test_the_same_batch_draws_other_masks():
    from train_gpt_b200.step import Trainer
    cfg = dataclasses.replace(_cfg(dropout=0.5), lr=0.0, weight_decay=0.0)
    for graph in (False, True):
        tr = Trainer(cfg, torch.device("cuda", 0), seed=3, graph=graph)
        batch = _batch(cfg, 0)
        assert len({float(tr.step(*batch)[0]) for _ in range(3)}) == 3
        with torch.no_grad():
            assert torch.equal(tr.model.loss(*batch), tr.model.loss(*batch))
        del tr


def test_a_plain_run_of_the_operators():
    """Without a model: one projection, heads as slices of it, attention, dropout into the stream, norm, gated feed-forward; gradients of every
    input against differences of the loss along a direction, in 64 bits with the same masks."""
    import block_reference as ref
    from train_gpt_b200 import kernels
    gen = torch.Generator(device="cuda").manual_seed(0)
    B, T, H, D, F = 2, 24, 2, 32, 96

    def rnd(*shape, std=1.0):
        return (std * torch.randn(shape, device="cuda", generator=gen)).to(torch.bfloat16)
    x, w_qkv, w_o, gamma = rnd(B, T, H * D), rnd(H * D, 3 * H * D, std=0.12), rnd(H * D, H * D, std=0.12), (1 + rnd(H * D, std=0.1))
    qs, ks, wg, wu = 1 + rnd(D, std=0.1), 1 + rnd(D, std=0.1), rnd(H * D, F, std=0.12), rnd(H * D, F, std=0.12)
    g = rnd(B, T, F)
    seed = torch.tensor([77], device="cuda")
    mask, scale = ref.kept(x.numel(), 0.25, 77, 4)
    mask = torch.from_numpy(mask).to("cuda").view(x.shape)
    at = torch.arange(T, device="cuda").expand(B, T)

    def attention(q, k, v):
        q, k, v = (t.transpose(1, 2) for t in (q, k, v))
        s = (q @ k.transpose(-1, -2)) / D ** 0.5 + torch.full((T, T), float("-inf"), device="cuda", dtype=q.dtype).triu(1)
        return (torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, H * D)

    def kernel(x, w_qkv, w_o, gamma, qs, ks, wg, wu):
        q, k, v = (t.unflatten(-1, (H, D)) for t in (x @ w_qkv).chunk(3, -1))
        q, k = kernels.qk_norm_rope(q, k, qs, ks, 1e-5)
        y = kernels.dropout(attention(q, k, v) @ w_o, 0.25, seed, 4, residual=x)
        return kernels.gated_linear(kernels.rms_norm(y, gamma, 1e-5), wg, wu)

    def plain(x, w_qkv, w_o, gamma, qs, ks, wg, wu):
        q, k, v = (t.unflatten(-1, (H, D)) for t in (x @ w_qkv).chunk(3, -1))
        q, k = (ref.rotate(ref.norm(t, w, 1e-5), at, 10000.0, D, False) for t, w in ((q, qs), (k, ks)))
        y = torch.where(mask, (attention(q, k, v) @ w_o) * scale, 0.0) + x
        n = ref.norm(y, gamma, 1e-5)
        return ref.act(n @ wg, "silu")[0] * (n @ wu)
    leaves = [t.detach().requires_grad_() for t in (x, w_qkv, w_o, gamma, qs, ks, wg, wu)]
    grads = torch.autograd.grad(kernel(*leaves), leaves, g)
    v = [t.detach().double() for t in leaves]
    for i, d in enumerate(grads):
        step = torch.randn(v[i].shape, device="cuda", dtype=torch.float64, generator=gen)
        ends = [(plain(*v[:i], v[i] + s * 1e-5 * step, *v[i + 1:]) * g.double()).sum() for s in (1, -1)]
        # some twenty bf16 roundings of 2^-8 one way and back, each of which reaches the result with about its share of the terms
        assert abs((ends[0] - ends[1]) / 2e-5 - (d.double() * step).sum()) <= 20 * ref.BF * float((d.double() * step).norm()) * 4, i

"""The edge cases of losses.capped_distillation in each form of its kernel, which rows and vocabulary choose.

  plain      no table of the cap                               few logits for a block
  short      a table that up to eight kept rows share          many rows of few logits
  one        a table, a kept row a block
  two        a table that two kept rows share
  unkept     a table, the row read again for the gradient      vocabularies that shared memory does not hold
  groups     the same, several rows a block
The loss alone (no gradient) has its own table, of exponentials, and keeps no row.  Temperatures choose how the second exponential is had: 1 none, 2
and 4 the first one squared once and twice, 3 its own.

Tolerances are those of test_gpu_distill.  A saturated logit's derivative of the cap is taken in 64 bits as 4 e / (1 + e)^2, e = exp(-2 |x| / c), which
1 - tanh^2 loses; in the kernels u = 2 / (1 + exp(2 |x| / c)) has an exponent of up to 88 rounded three times, 3 * 88 * 2^-24 of u, which
(4 DELTA + 2^-16) holds, and what is below 2^-126 may be 0: 2^-125 of the summands (u (2 - u) is at most twice that)."""
import math

import pytest
import torch

import operators_reference as ref
from test_gpu_distill import _check_distill, _delta, _log_tol, _logits, _teacher

pytestmark = pytest.mark.gpu
INF = math.inf
NAN = math.nan

FORMS = {"plain": (40, 2050), "short": (17003, 300), "one": (40, 20001), "two": (301, 50257), "unkept": (12, 130001), "groups": (301, 130001)}
forms = pytest.mark.parametrize("rows,vocab", list(FORMS.values()), ids=list(FORMS))
temperatures = pytest.mark.parametrize("t,w", [(1.0, 1.0), (2.0, 0.5), (4.0, 0.5), (3.0, 0.5)])


def _targets(rows, vocab, w):
    g = torch.Generator(device="cuda").manual_seed(rows)
    return torch.randint(0, vocab, (rows,), device="cuda", generator=g) if w < 1 else None


def _both(x, teacher, t, w, targets, cap=15.0):
    """(row losses, gradient, the row losses of the form without a gradient)"""
    from train_gpt_b200 import ops
    rows, d = ops.softcap_distill(x, *teacher, cap, targets, t, w)
    alone, none = ops.softcap_distill(x, *teacher, cap, targets, t, w, want_grad=False)
    assert none is None
    return rows, d, alone


@forms
@temperatures
def test_a_nan_anywhere_in_a_row(rows, vocab, t, w):
    """In each element of a piece, beside and on a named logit, at the row's ends, on the target: the whole row is NaN and no other row is touched."""
    x = _logits(rows, vocab, seed=31)
    ids, logp, rest = teacher = _teacher(rows, vocab, 9, 15.0, t)
    targets = _targets(rows, vocab, w)
    want = _both(x, teacher, t, w, targets)
    assert all(v.isfinite().all() for v in want)
    named = ids[:, 3].tolist()
    at = {r: 128 + (r - r * vocab) % 8 for r in range(8)}              # each element of a 16-byte piece, wherever the row begins
    at.update({8: named[8] - 1 if named[8] else 1, 9: 0, 10: vocab - 1, 11: named[11]})
    if rows > 20:
        for i in range(8):                                             # the other elements of a named logit's piece
            r = 12 + i
            at[r] = min(max((r * vocab + named[r]) // 8 * 8 + i - r * vocab, 0), vocab - 1)
        at[20] = int(targets[20]) if w < 1 else int(ids[20, 0])
        at[rows - 1] = 7
    bad = x.clone()
    for r, c in at.items():
        bad[r, c] = NAN
    got = _both(bad, teacher, t, w, targets)
    hit = torch.zeros(rows, dtype=torch.bool, device="cuda")
    hit[list(at)] = True
    for g, v in zip(got, want):
        assert g[hit].isnan().all(), [r for r in at if not g[r].isnan().all()]
        assert torch.equal(g[~hit], v[~hit])


def _exact(x, ids, logp, rest, cap, targets, t, w):
    """(the rows' losses, the gradient of their mean, the size of its summands), the cap's derivative as it is where it is far below 2^-53."""
    x = x.double()
    z = ref.capped(x, cap).requires_grad_()
    vocab = x.shape[1]
    logq = torch.log_softmax(z / t, -1)
    ids = ids.long()
    p = logp.double().exp()
    row = w * t * t * (p * (logp.double() - logq.gather(1, ids))).sum(-1)
    named = torch.zeros_like(x, dtype=torch.bool).scatter_(1, ids, True)
    r = rest.double()
    row = row + w * t * t * r.exp() * (r - logq.masked_fill(named, -INF).logsumexp(-1))
    if targets is not None:
        row = row - (1 - w) * torch.log_softmax(z, -1).gather(1, targets.unsqueeze(-1)).squeeze(-1)
    (dz,) = torch.autograd.grad(row.mean(), z)
    e = torch.exp(-2 * x.abs() / cap)
    sech2 = 4 * e / (1 + e) ** 2
    # the summands without their signs and without the cap's derivative
    q, q1 = torch.softmax(z.detach() / t, -1), torch.softmax(z.detach(), -1)
    tail = torch.where(named, 0.0, q).sum(-1, keepdim=True)
    size = w * t * (q * (p.sum(-1, keepdim=True) + r.exp().unsqueeze(-1) * (1 + torch.where(named, 0.0, 1 / tail))) + torch.zeros_like(x).scatter_add_(1, ids, p))
    if targets is not None:
        size = size + (1 - w) * (q1 + torch.zeros_like(x).scatter_(1, targets.unsqueeze(-1), 1.0))
    return row.detach(), dz * sech2, size / x.shape[0], sech2


@pytest.mark.parametrize("cap", [15.0, 8.0, 0.75])
@pytest.mark.parametrize("rows,vocab", [FORMS[f] for f in ("plain", "one", "two", "unkept")], ids=("plain", "one", "two", "unkept"))
@pytest.mark.parametrize("t,w", [(1.0, 1.0), (2.0, 0.5), (3.0, 0.5)])
def test_saturated_logits(rows, vocab, cap, t, w):
    """From where tanh is near 1 to far beyond it, both signs, in every element of a piece, on named logits and at the row's ends."""
    x = _logits(rows, vocab, seed=32).float() * (cap / 15)
    far = [cap * v for v in (4.0, 8.0, 11.0, 15.9, 16.1, 17.0, 18.0, 20.0, 25.0, 31.0, 33.0, 40.0, 44.0, 46.0, 63.0, 65.0, 130.0, 1e6)] + [3e38, INF]
    ids, logp, rest = _teacher(rows, vocab, 9, 15.0, t)
    targets = _targets(rows, vocab, w)
    r = torch.arange(rows, device="cuda")
    v = torch.tensor(far, device="cuda")[r % len(far)].unsqueeze(1)
    u = torch.tensor(far, device="cuda")[(r + 10) % len(far)].unsqueeze(1)
    x[:, 200:217], x[:, 300:317] = v, -u
    x[:, :1], x[:, vocab - 1:] = u, -v
    x.scatter_(1, ids[:, 2:3].long(), -v)
    x = x.to(torch.bfloat16)
    row, want, size, sech2 = _exact(x, ids, logp, rest, cap, targets, t, w)
    got_rows, got, alone = _both(x, (ids, logp, rest), t, w, targets, cap)
    delta = _delta(max(cap, 15.0), min(t, 1.0))
    bound = 2.0 ** -8 * want.abs() + (4 * delta + 2.0 ** -16) * size * sech2 + 2.0 ** -125 * size + 2.0 ** -133
    over = (got.double() - want).abs() / bound
    assert bool((over <= 1).all()), (float(over.max()), divmod(int(over.argmax()), vocab))
    tol = w * t * t * (_log_tol(cap, t) + 2.0 ** -18) + (1 - w) * _log_tol(cap, 1.0)
    assert float((got_rows.double() - row).abs().max()) <= tol and float((alone.double() - row).abs().max()) <= tol


@forms
@temperatures
def test_repeated_missing_and_empty_entries(rows, vocab, t, w):
    """One id for several entries, entries and targets outside the vocabulary with anything in their place, probabilities of 0, padded rows."""
    from train_gpt_b200 import losses
    ids, logp, rest = _teacher(rows, vocab, 12, 15.0, t)
    targets = _targets(rows, vocab, w)
    ids[0, 5] = ids[0, 2]
    ids[1, 1:] = ids[1, 0]
    ids[2, -1] = ids[2, 0]
    ids[3, 4] = -1
    ids[4, 0] = vocab
    ids[5, 3] = 2 ** 31 - 1
    logp[6, 3:] = -INF
    rest[7] = -INF
    pad = rows - max(1, rows // 8)
    ids[pad:] = -1
    rest[pad:] = 0
    if targets is not None:
        targets[0] = ids[0, 2].long()
        targets[1] = ids[1, 0].long()
        targets[8] = -100
        targets[9] = vocab
        targets[pad:] = -1
    x = _logits(rows, vocab, seed=33)
    loss, d = _check_distill(x, ids, logp, rest, 15.0, targets, t, w)
    assert not d[pad:].any()
    held = logp.masked_fill((ids < 0) | (ids >= vocab), NAN)
    leaf = x.clone().requires_grad_()
    again = losses.capped_distillation(leaf, losses.TopLogits(ids, held, rest), 15.0, target_ids=targets, temperature=t, weight=w)
    again.backward()
    assert torch.equal(again.detach(), loss) and torch.equal(leaf.grad, d)


@forms
@pytest.mark.parametrize("t,w", [(2.0, 0.5), (1.0, 1.0)])
def test_upstream_gradients_and_a_second_pass(rows, vocab, t, w):
    """An upstream gradient of a power of two gives the same digits; of 1 the launch in the backward pass does nothing; a second pass has its own memory."""
    from train_gpt_b200 import losses
    teacher = losses.TopLogits(*_teacher(rows, vocab, 8, 15.0, t))
    targets = _targets(rows, vocab, w)
    leaf = _logits(rows, vocab, seed=34).requires_grad_()

    def loss():
        return losses.capped_distillation(leaf, teacher, 15.0, target_ids=targets, temperature=t, weight=w)
    (one,) = torch.autograd.grad(loss(), leaf)
    up = loss()
    (a,) = torch.autograd.grad(up, leaf, torch.tensor(4.0, device="cuda"), retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(up, leaf, torch.tensor(1.0, device="cuda"))
    assert torch.equal(a, kept) and a.data_ptr() != b.data_ptr()
    assert torch.equal(b, one) and torch.equal(a, 4 * one)


@forms
def test_pitches_and_alignments(rows, vocab):
    """Rows of an even and of an odd pitch whose pad is NaN, and logits that begin off a 16-byte boundary, as contiguous ones."""
    teacher = _teacher(rows, vocab, 8, 15.0, 2.0)
    targets = _targets(rows, vocab, 0.5)
    x = _logits(rows, vocab, seed=35)
    want = _both(x, teacher, 2.0, 0.5, targets)
    for pitch in (vocab + 15, (vocab + 63) // 64 * 64):
        base = torch.full((rows, pitch), NAN, dtype=torch.bfloat16, device="cuda")
        base[:, :vocab] = x
        got = _both(base[:, :vocab], teacher, 2.0, 0.5, targets)
        for name, g, v in zip(("rows", "gradient", "rows alone"), got, want):
            # (a row's order of additions goes by its alignment, which the pitch changes: the last bits of its sums)
            tol = 4 * 0.5 * (_log_tol(15.0, 2.0) + 2.0 ** -18) + 0.5 * _log_tol(15.0, 1.0)
            if name != "gradient":
                assert float((g - v).abs().max()) <= tol
            else:
                size = ref.distill_scale(x, *teacher, 15.0, targets, 2.0, 0.5)
                assert bool(((g.double() - v.double()).abs() <= 2 * (2.0 ** -8 * v.double().abs() + (4 * _delta(15.0, 1.0) + 2.0 ** -16) * size) + 2.0 ** -133).all())
                del size
        del base, got
    for shift in (1, 6):
        flat = torch.empty(rows * vocab + shift, dtype=torch.bfloat16, device="cuda")
        flat[shift:] = x.reshape(-1)
        got = _both(flat[shift:].view(rows, vocab), teacher, 2.0, 0.5, targets)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert float((got[2] - want[2]).abs().max()) <= tol


def test_gradient_rows_between_the_logits_rows():
    """One buffer of twice the pitch, the gradient's rows between the logits': allowed by the C entry, and the same bits."""
    import ctypes
    from train_gpt_b200 import _lib, ops
    rows, vocab, ld = 40, 1000, 2048
    ids, logp, rest = _teacher(rows, vocab, 8, 15.0, 2.0)
    x = _logits(rows, vocab, seed=36)
    base = torch.zeros(rows, ld, dtype=torch.bfloat16, device="cuda")
    base[:, :vocab] = x
    out = base[:, 1024:1024 + vocab]
    row_loss = torch.empty(rows, device="cuda")
    a = _lib.DistillArgs(logits=base.data_ptr(), ids=ids.data_ptr(), logp=logp.data_ptr(), log_rest=rest.data_ptr(), cap=15.0, temperature=2.0, weight=1.0,
                         dlogits=out.data_ptr(), row_loss=row_loss.data_ptr(), rows=rows, vocab=vocab, ld=ld, k=8)
    assert _lib.load().tg_softcap_distill(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.TG_OK
    view = torch.zeros(rows, ld, dtype=torch.bfloat16, device="cuda")
    view[:, :vocab] = x
    want_rows, want = ops.softcap_distill(view[:, :vocab], ids, logp, rest, 15.0, None, 2.0, 1.0)
    assert torch.equal(row_loss, want_rows) and torch.equal(out, want) and torch.equal(base[:, :vocab], x)
    assert not base[:, vocab:1024].any() and not base[:, 1024 + vocab:].any()


@pytest.mark.parametrize("vocab", [16399, 16400, 16401])
def test_top_logits_around_the_first_sampled_length(vocab):
    """Rows of the length from which the first bound comes from a sample, and of one less: the largest logits only in what a sample sees, only elsewhere,
    anywhere."""
    from test_gpu_distill import _check_top
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(24, vocab, device="cuda", generator=g)
    start = torch.arange(24, device="cuda").unsqueeze(1) * vocab
    piece = (torch.arange(vocab, device="cuda").unsqueeze(0) - (-start) % 8) // 8
    seen = (piece >= 0) & (piece % 64 < 8)
    big = 3 + 3 * torch.rand(24, vocab, device="cuda", generator=g)
    few = torch.rand(24, vocab, device="cuda", generator=g) < 300 / vocab
    kind = torch.arange(24, device="cuda").unsqueeze(1) // 8
    x = torch.where(torch.where(kind == 0, ~seen & few, torch.where(kind == 1, seen, few)), big, x).to(torch.bfloat16)
    for k in (1, 64, 65, 256):
        _check_top(x, 15.0, k, 1.0)

"""losses.top_logits and losses.capped_distillation against their 64-bit forms.

Tolerances.  Capped logits over T come from u = 2 / (1 + exp(2 |x| / c)), three approximations of 2^-22 of themselves and a few roundings of
2^-24, so that z / T is off by at most (c / T) 2^-20 and exp of it by DELTA = (c / T) 2^-20 + 2^-21 of itself.  Sums of such terms are off by as
much and by the additions' 2^-24 each over the depth of the sum (below 2^8).  A log-probability is off by twice that and by the rounding
of numbers up to 2 c / T + 17.  A gradient's element is rounded to bf16 once, 2^-8 of it, after errors of 4 DELTA + 2^-16 of its summands; below
2^-126 bf16's numbers lie 2^-133 apart, so that half of that is lost there whatever the element (at a cap of 64 elements reach 2^-180)."""
import math

import pytest
import torch

import operators_reference as ref

pytestmark = pytest.mark.gpu
INF = math.inf


def _delta(cap, t):
    return cap / t * 2.0 ** -20 + 2.0 ** -21


def _logits(rows, vocab, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = scale * torch.randn(rows, vocab, device="cuda", generator=g)
    x[:, :: max(1, vocab // 5)] += 9
    return x.to(torch.bfloat16)


def _log_tol(cap, t):
    return 2 * _delta(cap, t) + 2.0 ** -15 + (2 * cap / t + 17) * 2.0 ** -22


def _check_top(x, cap, k, t):
    from train_gpt_b200 import losses
    top = losses.top_logits(x, cap, k, temperature=t)
    vocab = x.shape[-1]
    ids, logp, rest = ref.top_logits(x.reshape(-1, vocab).double(), cap, k, t)
    assert top.ids.dtype == torch.int32 and top.ids.shape == (*x.shape[:-1], k)
    assert torch.equal(top.ids.reshape(-1, k).long(), ids)
    tol = _log_tol(cap, t)
    assert float((top.logp.reshape(-1, k).double() - logp).abs().max()) <= tol
    got = top.log_rest.reshape(-1).double()
    assert torch.equal(got == -INF, rest == -INF)
    fin = rest > -INF
    # (near 0 it comes from the smaller part, so that it keeps its relative precision)
    assert bool(((got - rest).abs()[fin] <= tol * torch.clamp(rest[fin].abs(), max=1.0) + 2.0 ** -22).all())
    return top


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 7), (2, 8, 3), (5, 9, 1), (40, 250, 16), (300, 256, 8), (17, 256, 256), (64, 1000, 256), (9, 4097, 100), (33, 32000, 64),
                                          (4, 50257, 64), (300, 50257, 256), (2, 50304, 1), (2, 70001, 200), (3, 120001, 64), (1, 300000, 256)])
@pytest.mark.parametrize("cap,t", [(15.0, 1.0), (30.0, 4.0)])
def test_top_logits(rows, vocab, k, cap, t):
    _check_top(_logits(rows, vocab, seed=rows + vocab), cap, k, t)


def test_top_logits_of_equal_sorted_and_crowded_rows():
    """Rows that the first bound does not thin out: all logits equal, sorted ones, the largest side by side, two values only, +-0."""
    vocab = 20011
    x = torch.zeros(8, vocab, device="cuda")
    x[1] = torch.arange(vocab, device="cuda") / 1000
    x[2] = -torch.arange(vocab, device="cuda") / 1000
    x[3, 7000:7400] = torch.linspace(5, 9, 400, device="cuda")
    x[4, 1::2] = 1
    x[5, ::3] = -0.0
    x[6] = -INF
    x[6, 17] = 1
    x[7, -130:] = 2
    for k in (1, 64, 255):
        _check_top(x.to(torch.bfloat16), 15.0, k, 1.0)
    wide = torch.full((2, 130001), 0.5, device="cuda", dtype=torch.bfloat16)
    wide[1, -1] = 3
    _check_top(wide, 15.0, 100, 1.0)


@pytest.mark.parametrize("vocab", [16416, 50257, 140001])
def test_top_logits_where_a_sample_of_the_row_misleads(vocab):
    """The bound comes from eight 16-byte pieces of every 64 of a long row: the largest logits all in the others, all in those, or in one of the two
    in so small a number that the bound lets too few through."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(6, vocab, device="cuda", generator=g)
    start = torch.arange(6, device="cuda").unsqueeze(1) * vocab                 # (a row's own pieces begin at the next 16-byte boundary)
    piece = (torch.arange(vocab, device="cuda").unsqueeze(0) - (-start) % 8) // 8
    seen = (piece >= 0) & (piece % 64 < 8)
    big = 3 + 3 * torch.rand(6, vocab, device="cuda", generator=g)
    few = torch.rand(6, vocab, device="cuda", generator=g) < 400 / vocab
    x = torch.where(torch.stack([~seen[0], seen[1], ~seen[2] & few[2], seen[3] & few[3], few[4], torch.zeros_like(few[5])]), big, x)
    x[5] = torch.where(seen[5], x[5], -20.0)
    for k in (1, 33, 64, 65, 256):
        _check_top(x.to(torch.bfloat16), 15.0, k, 1.0)


@pytest.mark.parametrize("vocab", [4099, 30000])
def test_top_logits_on_a_coarse_grid(vocab):
    """Hundreds of logits equal to the k-th, above and below 0, with and without a NaN."""
    from train_gpt_b200 import losses
    g = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(5, vocab, device="cuda", generator=g)
    x = torch.stack([1 + 0.02 * x[0], -1 + 0.02 * x[1], (2 * x[2]).round(), 64 + x[3], -x[4].abs().round()]).to(torch.bfloat16)
    for k in (1, 7, 64, 256):
        _check_top(x, 15.0, k, 1.0)
    x[:, vocab // 2] = float("nan")
    top = losses.top_logits(x, 15.0, 64)
    x[:, vocab // 2] = INF
    ids = ref.top_logits(x.double(), 15.0, 64, 1.0)[0]
    assert torch.equal(top.ids.long(), ids) and bool(top.logp.isnan().all())


@pytest.mark.parametrize("rows,vocab,k", [(160, 40001, 16), (320, 33000, 64), (700, 20000, 200), (1200, 5000, 20), (1190, 1500, 100), (1300, 4095, 256), (600, 9001, 8)])
def test_top_logits_of_more_rows_than_fit(rows, vocab, k):
    """Several rows at a time on an SM, with one or two groups of threads left without a row in the last round."""
    _check_top(_logits(rows, vocab, seed=rows), 15.0, k, 1.0)


@pytest.mark.parametrize("cap,t", [(64.0, 1.0), (2.0 ** -10, 1.0), (1.0, 1024.0), (2.0, 0.03125), (11.0, 3.0)])
def test_the_range_of_caps_and_temperatures(cap, t):
    """Logits in proportion to the cap, so that tanh is far from its ends and at them."""
    x = (_logits(40, 5003, seed=11).float() * (cap / 15)).to(torch.bfloat16)
    top = _check_top(x, cap, 40, t)
    targets = torch.randint(0, 5003, (40,), device="cuda")
    _check_distill((_logits(40, 5003, seed=12).float() * (cap / 15)).to(torch.bfloat16), top.ids, top.logp, top.log_rest, cap, targets, t, 0.25)
    if cap <= 64 * t:
        _check_distill((_logits(170, 20001, seed=13).float() * (cap / 15)).to(torch.bfloat16), *_check_top((_logits(170, 20001, seed=14).float() * (cap / 15)).to(torch.bfloat16), cap, 8, t),
                       cap, None, t, 1.0)


def test_the_largest_vocabulary():
    vocab = 1 << 20
    x = _logits(3, vocab, seed=15)
    top = _check_top(x, 15.0, 100, 2.0)
    targets = torch.tensor([vocab - 1, 5, vocab], device="cuda")
    _check_distill(_logits(3, vocab, seed=16), top.ids, top.logp, top.log_rest, 15.0, targets, 2.0, 0.5)


def test_top_logits_with_infinities_and_nan():
    from train_gpt_b200 import losses
    x = _logits(4, 5003, seed=2)
    x[0, 11] = INF
    x[0, 4000] = INF
    x[1, ::2] = -INF
    _check_top(x[:2], 15.0, 20, 2.0)
    x[2, 77] = float("nan")
    top = losses.top_logits(x, 15.0, 20)
    assert top.ids[2, 0] == 77 and top.logp[2].isnan().all() and top.log_rest[2].isnan()
    assert not top.logp[3].isnan().any() and len(set(top.ids[2].tolist())) == 20


def test_top_logits_views_shapes_and_streams():
    """A slice of a padded vocabulary whose pad is NaN, rows at every alignment, a batch of sequences, another stream, a replayed graph."""
    from train_gpt_b200 import losses
    base = torch.full((6, 5, 2064), float("nan"), dtype=torch.bfloat16, device="cuda")
    base[..., 3:2050] = _logits(30, 2047, seed=4).view(6, 5, 2047)
    view = base[..., 3:2050]
    want = _check_top(view, 15.0, 31, 1.0)
    same = losses.top_logits(view.contiguous(), 15.0, 31)
    assert torch.equal(want.ids, same.ids)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = losses.top_logits(view, 15.0, 31)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = losses.top_logits(view, 15.0, 31)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    odd = torch.randn(2047 * 9, device="cuda").to(torch.bfloat16)
    for shift in range(1, 8):
        _check_top(odd[shift:shift + 4 * 2047].view(4, 2047), 15.0, 9, 1.0)
    assert losses.top_logits(view[:0], 15.0, 31).ids.shape == (0, 5, 31)


def test_top_logits_twice_the_same_bits():
    x = _logits(600, 50257, seed=9)
    from train_gpt_b200 import losses
    a = losses.top_logits(x, 15.0, 256)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(a, losses.top_logits(x, 15.0, 256)))


# ---- the student's loss ----------------------------------------------------------------------------------------------

def _teacher(rows, vocab, k, cap, t, seed=1, rest=True, ids_dtype=torch.int32):
    z = ref.capped(_logits(rows, vocab, seed=seed).double(), cap) / t
    logq = torch.log_softmax(z, -1)
    logp, ids = torch.topk(logq, k)
    if rest:
        return ids.to(ids_dtype), logp.float(), logq.scatter(1, ids, -INF).logsumexp(-1).float()
    return ids.to(ids_dtype), torch.log_softmax(logp, -1).float(), None


def _check_distill(x, ids, logp, rest, cap, targets, t, w, mass=1.0):
    from train_gpt_b200 import losses, ops
    vocab = x.shape[-1]
    flat = lambda v: None if v is None else v.flatten(0, -2)      # noqa: E731
    row, d = ref.distill(x.detach().reshape(-1, vocab), flat(ids), flat(logp), None if rest is None else rest.reshape(-1), cap,
                         None if targets is None else targets.reshape(-1), t, w)
    size = ref.distill_scale(x.detach().reshape(-1, vocab), flat(ids), flat(logp), None if rest is None else rest.reshape(-1), cap,
                             None if targets is None else targets.reshape(-1), t, w)
    leaf = x.detach().requires_grad_()
    loss = losses.capped_distillation(leaf, losses.TopLogits(ids, logp, rest), cap, target_ids=targets, temperature=t, weight=w)
    (got,) = torch.autograd.grad(loss, leaf)
    tol = w * t * t * mass * (_log_tol(cap, t) + 2.0 ** -18) + (1 - w) * _log_tol(cap, 1.0)
    rows, dd = ops.softcap_distill(x.detach(), ids, logp, rest, cap, targets, t, w)
    assert torch.equal(dd, got)
    fin = row.isfinite()
    assert torch.equal(rows.reshape(-1).isfinite(), fin)
    assert float((rows.reshape(-1).double() - row)[fin].abs().max()) <= tol
    if bool(fin.all()):
        assert abs(float(loss.detach()) - float(row.mean())) <= tol
    bound = 2.0 ** -8 * d.abs() + (4 * _delta(cap, min(t, 1.0)) + 2.0 ** -16) * size + 2.0 ** -133
    off = (got.reshape(-1, vocab).double() - d).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    with torch.no_grad():
        again = losses.capped_distillation(x.detach(), losses.TopLogits(ids, logp, rest), cap, target_ids=targets, temperature=t, weight=w)
    assert abs(float(again) - float(loss.detach())) <= tol
    return loss.detach(), got


@pytest.mark.parametrize("rows,vocab,k", [(1, 2, 1), (3, 9, 4), (2, 8, 8), (128, 256, 8), (40, 250, 250), (17, 1000, 33), (5, 4097, 256), (6, 50257, 64), (310, 50304, 32), (3, 120001, 64)])
@pytest.mark.parametrize("cap,t,w,rest", [(15.0, 1.0, 1.0, True), (15.0, 2.0, 0.5, True), (30.0, 1.0, 0.9, False), (30.0, 4.0, 1.0, False), (15.0, 2.0, 0.0, True)])
def test_distillation(rows, vocab, k, cap, t, w, rest):
    ids, logp, log_rest = _teacher(rows, vocab, k, cap, t, rest=rest and k < vocab, ids_dtype=torch.int64 if rows % 2 else torch.int32)
    targets = torch.randint(0, vocab, (rows,), device="cuda", dtype=torch.int32 if rows % 2 else torch.int64)
    targets[::2] = ids[::2, 0].to(targets.dtype)                             # some of them named by the teacher
    _check_distill(_logits(rows, vocab, seed=7), ids, logp, log_rest, cap, targets if w < 1 else None, t, w)


@pytest.mark.parametrize("rows,vocab,k,t,w", [(450, 9001, 130, 1.0, 1.0), (1201, 5000, 8, 2.0, 0.5), (700, 30001, 64, 4.0, 0.5), (330, 130000, 20, 3.0, 0.5), (1190, 300, 100, 1.0, 0.5), (12001, 300, 20, 2.0, 0.5), (5003, 1024, 70, 1.0, 1.0), (9001, 777, 5, 3.0, 0.5)])
def test_distillation_of_more_rows_than_fit(rows, vocab, k, t, w):
    """Rows beside each other on an SM (two that share a table, up to eight that are not kept), the last round not full."""
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, t)
    targets = torch.randint(0, vocab, (rows,), device="cuda") if w < 1 else None
    _check_distill(_logits(rows, vocab, seed=8), ids, logp, rest, 15.0, targets, t, w)


def test_missing_entries_padding_and_what_they_hold():
    """Entries and targets outside the vocabulary take no part, whatever stands at them; a padded row adds nothing and has no gradient."""
    rows, vocab, k = 24, 3001, 12
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 2.0)
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    ids[::3, 4] = -1
    ids[1::3, 0] = vocab
    ids[2, 3] = 2 ** 31 - 1
    ids[20:] = -1
    targets[5] = -100
    targets[6] = vocab
    targets[20:] = -1
    rest[20:] = 0
    x = _logits(rows, vocab, seed=3)
    loss, d = _check_distill(x, ids, logp, rest, 15.0, targets, 2.0, 0.5)
    assert not d[20:].any()
    gone = (ids < 0) | (ids >= vocab)
    for junk in (float("nan"), INF, -INF):
        held = logp.masked_fill(gone, junk)
        from train_gpt_b200 import losses
        leaf = x.clone().requires_grad_()
        again = losses.capped_distillation(leaf, losses.TopLogits(ids, held, rest), 15.0, target_ids=targets, temperature=2.0, weight=0.5)
        again.backward()
        assert torch.equal(again.detach(), loss) and torch.equal(leaf.grad, d)


def test_zero_probabilities_and_unnormalised_ones():
    rows, vocab, k = 6, 515, 10
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 1.0)
    logp[0, 3:] = -INF
    rest[1] = -INF
    rest[2] = 1.0                                                           # e of it: a row whose probabilities do not sum to one
    logp[3] += 0.5
    _check_distill(_logits(rows, vocab, seed=3), ids, logp, rest, 15.0, None, 1.0, 1.0, mass=4.5)
    none = torch.empty(rows, 0, dtype=torch.int32, device="cuda")           # no entries at all: the rest is everything
    _check_distill(_logits(rows, vocab, seed=3), none, torch.empty(rows, 0, device="cuda"), torch.zeros(rows, device="cuda"), 15.0, None, 1.0, 1.0)


def test_rest_without_a_tail_is_infinite():
    """The teacher names the whole vocabulary and still leaves something for the others."""
    from train_gpt_b200 import losses
    ids = torch.arange(16, device="cuda").expand(3, 16).contiguous()
    logp = torch.full((3, 16), math.log(1 / 32), device="cuda")
    x = _logits(3, 16)
    assert float(losses.capped_distillation(x, losses.TopLogits(ids, logp, torch.full((3,), math.log(0.5), device="cuda")), 15.0)) == INF
    assert math.isfinite(float(losses.capped_distillation(x, losses.TopLogits(ids, logp, torch.full((3,), -INF, device="cuda")), 15.0)))


def test_an_id_named_twice():
    rows, vocab, k = 9, 777, 40
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 2.0)
    ids[0, 5] = ids[0, 2]
    ids[1, 1:] = ids[1, 0]
    ids[2, -1] = ids[2, 0]
    targets = ids[:, 0].long().clone()
    x = _logits(rows, vocab, seed=5)
    a = _check_distill(x, ids, logp, rest, 15.0, targets, 2.0, 0.5)
    for _ in range(5):
        b = _check_distill(x, ids, logp, rest, 15.0, targets, 2.0, 0.5)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_infinite_and_nan_logits():
    from train_gpt_b200 import losses
    rows, vocab, k = 5, 2050, 16
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 1.0)
    x = _logits(rows, vocab, seed=5)
    x[0, 3], x[0, 9] = INF, -INF
    x[1, ids[1, 0].long()] = INF
    x[2, ids[2, 1].long()] = -INF
    _check_distill(x, ids, logp, rest, 15.0, ids[:, 1].long(), 1.0, 0.5)
    x[3, 100] = float("nan")
    x[4, ids[4, 0].long()] = float("nan")
    leaf = x.clone().requires_grad_()
    losses.capped_distillation(leaf, losses.TopLogits(ids, logp, rest), 15.0).backward()
    assert leaf.grad[3].isnan().all() and leaf.grad[4].isnan().all() and leaf.grad[:3].isfinite().all()


@pytest.mark.parametrize("scale", [1.0, 0.125, 3.0])
def test_upstream_gradient_and_repeated_backward(scale):
    """An upstream gradient other than one makes the gradient again, rounded once; the node can be used twice with retain_graph."""
    from train_gpt_b200 import losses
    rows, vocab, k = 33, 1030, 8
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 2.0)
    x = _logits(rows, vocab, seed=5)
    _, d1 = _check_distill(x, ids, logp, rest, 15.0, None, 2.0, 1.0)
    leaf = x.clone().requires_grad_()
    loss = losses.capped_distillation(leaf, losses.TopLogits(ids, logp, rest), 15.0, temperature=2.0)
    (a,) = torch.autograd.grad(loss, leaf, torch.tensor(scale, device="cuda"), retain_graph=True)
    kept = a.clone()
    (b,) = torch.autograd.grad(loss, leaf, torch.tensor(scale, device="cuda"))
    assert torch.equal(a, b) and torch.equal(a, kept) and a.data_ptr() != b.data_ptr()
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(loss, leaf)
    if scale in (1.0, 0.125):                                                # powers of two: the same digits
        assert torch.equal(a, (d1.float() * scale).to(torch.bfloat16))
    _, want = ref.distill(x, ids, logp, rest, 15.0, None, 2.0, 1.0)
    size = ref.distill_scale(x, ids, logp, rest, 15.0, None, 2.0, 1.0)
    assert bool(((a.double() - scale * want).abs() <= scale * (2.0 ** -8 * want.abs() + (4 * _delta(15.0, 1.0) + 2.0 ** -16) * size)).all())


def test_overwritten_inputs_scale_the_gradient_at_hand():
    from train_gpt_b200 import losses
    ids, logp, rest = _teacher(7, 300, 8, 15.0, 2.0)
    x = _logits(7, 300, seed=5)
    for which in range(2):
        leaf = x.clone().requires_grad_()
        t = losses.TopLogits(ids.clone(), logp.clone(), rest)
        loss = losses.capped_distillation(leaf, t, 15.0)
        (want,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        loss = losses.capped_distillation(leaf, t, 15.0)
        with torch.no_grad():
            (t.ids, t.logp)[which].zero_()
        (got,) = torch.autograd.grad(loss, leaf, torch.tensor(2.0, device="cuda"))
        assert torch.equal(got, 2 * want)
        # the gradient at hand has gone to the caller, or there is nothing to make another from
        t = losses.TopLogits(ids.clone(), logp.clone(), rest)
        loss = losses.capped_distillation(leaf, t, 15.0)
        torch.autograd.grad(loss, leaf, retain_graph=True)
        with torch.no_grad():
            (t.ids, t.logp)[which].zero_()
        with pytest.raises(RuntimeError, match="overwritten"):
            torch.autograd.grad(loss, leaf)


def test_one_row_for_many():
    """Expanded logits, whose rows lie on one another, at every axis."""
    from train_gpt_b200 import losses
    row = _logits(1, 777, seed=21)
    ids, logp, rest = _teacher(6, 777, 8, 15.0, 1.0)
    for x in (row.expand(6, 777), row.view(1, 1, 777).expand(2, 3, 777), _logits(3, 777, seed=22).expand(2, 3, 777), _logits(2, 777, seed=23).view(2, 1, 777).expand(2, 3, 777)):
        _check_top(x, 15.0, 20, 1.0)
        lead = x.shape[:-1]
        t = losses.TopLogits(ids.view(*lead, 8), logp.view(*lead, 8), rest.view(lead))
        leaf = x.clone().requires_grad_()
        want = losses.capped_distillation(leaf, t, 15.0)
        want.backward()
        base = x.detach().requires_grad_()
        got = losses.capped_distillation(base, t, 15.0)
        (d,) = torch.autograd.grad(got, base)
        assert torch.equal(got.detach(), want.detach()) and torch.equal(d, leaf.grad)


def test_a_teacher_that_names_nothing():
    """No entries: all of its probability is the rest's."""
    from train_gpt_b200 import losses
    x = _logits(5, 301, seed=24)
    ids, logp, rest = torch.zeros(5, 0, dtype=torch.int32, device="cuda"), torch.zeros(5, 0, device="cuda"), torch.zeros(5, device="cuda")
    leaf = x.clone().requires_grad_()
    loss = losses.capped_distillation(leaf, losses.TopLogits(ids, logp, rest), 15.0, target_ids=torch.arange(5, device="cuda"), weight=0.5)
    loss.backward()
    hard = x.clone().requires_grad_()
    want = losses.capped_distillation(hard, losses.TopLogits(ids, logp, rest), 15.0, target_ids=torch.arange(5, device="cuda"), weight=0.0)
    want.backward()
    # its own rest is all there is, so that only the targets' half is left
    assert abs(float(loss.detach()) - 0.5 * float(want.detach())) <= _log_tol(15.0, 1.0)
    assert float((leaf.grad.double() - 0.5 * hard.grad.double()).abs().max()) <= 2.0 ** -8 * 0.5 / 5 + (4 * _delta(15.0, 1.0) + 2.0 ** -16) * 2 / 5


def test_second_derivatives_are_an_error():
    from train_gpt_b200 import losses
    ids, logp, rest = _teacher(3, 300, 8, 15.0, 2.0)
    leaf = _logits(3, 300).requires_grad_()
    loss = losses.capped_distillation(leaf, losses.TopLogits(ids, logp, rest), 15.0)
    up = torch.ones((), device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(loss, leaf, up, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        d.float().sum().backward()


def test_views_shapes_and_graphs():
    """A padded vocabulary read in place (its pad is NaN), a batch of sequences, rows off the 16-byte boundary, a capture with its backward
    pass replayed on other data."""
    from train_gpt_b200 import losses
    b, s, vocab, k = 3, 5, 1001, 9
    ids, logp, rest = (v.view(b, s, *v.shape[1:]) for v in _teacher(b * s, vocab, k, 15.0, 2.0))
    targets = torch.randint(0, vocab, (b, s), device="cuda")
    base = torch.full((b, s, 1008), float("nan"), dtype=torch.bfloat16, device="cuda")
    x = _logits(b * s, vocab, seed=5).view(b, s, vocab)
    base[..., :vocab] = x
    plain = _check_distill(x, ids, logp, rest, 15.0, targets, 2.0, 0.5)
    sliced = _check_distill(base[..., :vocab], ids, logp, rest, 15.0, targets, 2.0, 0.5)
    assert torch.equal(plain[1], sliced[1]) and torch.equal(plain[0], sliced[0])
    shifted = torch.empty(b * s * vocab + 3, dtype=torch.bfloat16, device="cuda")
    shifted[3:] = x.reshape(-1)
    moved = _check_distill(shifted[3:].view(b, s, vocab), ids, logp, rest, 15.0, targets, 2.0, 0.5)
    assert torch.equal(plain[1], moved[1])
    leaf = x.clone().requires_grad_()
    teacher = losses.TopLogits(ids, logp, rest)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(losses.capped_distillation(leaf, teacher, 15.0, targets, 2.0, 0.5), leaf)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        loss = losses.capped_distillation(leaf, teacher, 15.0, targets, 2.0, 0.5)
        (d,) = torch.autograd.grad(loss, leaf)
    with torch.no_grad():
        leaf.copy_(x.flip(0))
    graph.replay()
    want = _check_distill(x.flip(0).contiguous(), ids, logp, rest, 15.0, targets, 2.0, 0.5)
    assert torch.equal(loss.detach(), want[0]) and torch.equal(d, want[1])


def test_no_rows():
    from train_gpt_b200 import losses
    leaf = torch.zeros(0, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    t = losses.TopLogits(torch.zeros(0, 4, dtype=torch.int32, device="cuda"), torch.zeros(0, 4, device="cuda"))
    loss = losses.capped_distillation(leaf, t, 15.0)
    loss.backward()
    assert loss.isnan() and leaf.grad.shape == (0, 64)


def test_against_differences():
    """The 64-bit loss along random directions against the kernel's gradient."""
    rows, vocab, k = 8, 260, 12
    ids, logp, rest = _teacher(rows, vocab, k, 15.0, 2.0)
    targets = torch.randint(0, vocab, (rows,), device="cuda")
    x = _logits(rows, vocab, seed=11)
    _, d = _check_distill(x, ids, logp, rest, 15.0, targets, 2.0, 0.5)
    g = torch.Generator(device="cuda").manual_seed(0)
    for _ in range(4):
        v = torch.randn(rows, vocab, device="cuda", dtype=torch.float64, generator=g)
        f = lambda e: float(ref.distill_rows(x.double() + e * v, ids, logp, rest, 15.0, targets, 2.0, 0.5).mean())   # noqa: E731
        diff = (f(1e-5) - f(-1e-5)) / 2e-5
        assert abs(diff - float((d.double() * v).sum())) <= 2.0 ** -7 * float((d.double() * v).abs().sum())


def test_agrees_with_the_capped_cross_entropy():
    """weight 0 is that loss up to the bf16 roundings of its capped logits: 2^-8 of |z| <= cap in three steps."""
    from train_gpt_b200 import losses
    x = _logits(50, 1000, seed=4)
    targets = torch.randint(0, 1000, (50,), device="cuda")
    none = losses.TopLogits(torch.empty(50, 0, dtype=torch.int32, device="cuda"), torch.empty(50, 0, device="cuda"))
    a = losses.capped_distillation(x, none, 15.0, targets, weight=0.0)
    assert abs(float(a) - float(losses.capped_cross_entropy(x, targets, 15.0))) <= 2 * 3 * 15 * 2.0 ** -8


def test_teacher_to_student():
    """A run as it is used: the teacher's top logits straight into the student's loss; a student equal to its teacher has loss 0 and no gradient."""
    from train_gpt_b200 import losses
    x = _logits(64, 2003, seed=8)
    t = losses.top_logits(x, 15.0, 32, temperature=2.0)
    leaf = x.clone().requires_grad_()
    loss = losses.capped_distillation(leaf, t, 15.0, temperature=2.0)
    loss.backward()
    assert abs(float(loss.detach())) <= 4 * (_log_tol(15.0, 2.0) + 2.0 ** -18)
    size = ref.distill_scale(x, t.ids, t.logp, t.log_rest, 15.0, None, 2.0, 1.0)
    assert bool((leaf.grad.double().abs() <= 4 * (4 * _delta(15.0, 1.0) + 2.0 ** -16) * size).all())

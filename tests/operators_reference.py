"""Plain 64-bit forms of the distillation operators and of the sandwich norm, for the tests that hold the kernels to them."""
import math

import torch

INF = math.inf


def capped(x, cap):
    return cap * torch.tanh(x / cap)


def top_logits(x, cap, k, t):
    """x float64 (R, V) holding bf16 values.  (ids, logp, log_rest); ties by the lower id, -0 is 0, NaN above all."""
    order = torch.where(x.isnan(), torch.full_like(x, INF), x + 0.0)
    nan = x.isnan().double()
    # NaN above +inf: sort by (is NaN, value), stable
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices
    ids = ids.gather(1, torch.sort(nan.gather(1, ids), dim=-1, descending=True, stable=True).indices)[:, :k]
    logq = torch.log_softmax(capped(x, cap) / t, -1)
    return ids, logq.gather(1, ids), logq.scatter(1, ids, -INF).logsumexp(-1)


def distill_rows(x, ids, logp, log_rest, cap, targets, t, w):
    """The rows' losses (R,), differentiable in x (float64)."""
    vocab = x.shape[1]
    z = capped(x, cap)
    logq = torch.log_softmax(z / t, -1)
    ids = ids.long()
    there = (ids >= 0) & (ids < vocab)
    lp = logp.double().masked_fill(~there, -INF)
    p = lp.exp()
    seen = logq.gather(1, ids.masked_fill(~there, 0))
    row = w * t * t * torch.where(p > 0, p * (lp.masked_fill(~(p > 0), 0.0) - seen), 0.0).sum(-1)
    if log_rest is not None:
        named = torch.zeros(x.shape[0], vocab + 1, dtype=torch.bool, device=x.device).scatter_(1, ids.masked_fill(~there, vocab), True)[:, :vocab]
        rest = log_rest.double()
        has = rest > -INF
        full = named.all(-1, keepdim=True)                       # (a logsumexp over nothing has no gradient)
        tail = torch.where(full, 0.0, logq.masked_fill(named & ~full, -INF)).logsumexp(-1)
        tail = torch.where(full.squeeze(-1), -INF, tail)
        row = row + w * t * t * torch.where(has, rest.exp() * (rest.masked_fill(~has, 0.0) - torch.where(has, tail, 0.0)), 0.0)
    if targets is not None and w < 1:
        targets = targets.long()
        ok = (targets >= 0) & (targets < vocab)
        ce = -torch.log_softmax(z, -1).gather(1, targets.masked_fill(~ok, 0).unsqueeze(-1)).squeeze(-1)
        row = row + (1 - w) * torch.where(ok, ce, 0.0)
    return row


def distill(x, ids, logp, log_rest, cap, targets, t, w):
    """(row losses, gradient of their mean)."""
    x = x.detach().double().requires_grad_()
    row = distill_rows(x, ids, logp, log_rest, cap, targets, t, w)
    (d,) = torch.autograd.grad(row.mean(), x)
    return row.detach(), d


def distill_scale(x, ids, logp, log_rest, cap, targets, t, w):
    """What the summands of a gradient's element amount to without their signs: (R, V)."""
    x = x.double()
    vocab = x.shape[1]
    z = capped(x, cap)
    q, q1 = torch.softmax(z / t, -1), torch.softmax(z, -1)
    ids = ids.long()
    there = (ids >= 0) & (ids < vocab)
    p = torch.where(there, logp.double().exp(), 0.0)
    at = ids.masked_fill(~there, vocab)
    wide = torch.zeros(x.shape[0], vocab + 1, dtype=torch.float64, device=x.device)
    mass = wide.clone().scatter_add_(1, at, p)[:, :vocab]
    named = wide.clone().scatter_(1, at, 1.0)[:, :vocab] > 0
    total, off = p.sum(-1, keepdim=True), 0.0
    if log_rest is not None:
        rest = log_rest.double().exp().unsqueeze(-1)
        tail = torch.where(named, 0.0, q).sum(-1, keepdim=True)
        off = torch.where(tail > 0, rest / tail, 0.0)
        total = total + rest
    s = w * t * (q * (total + torch.where(named, 0.0, off * torch.ones_like(q))) + mass)
    if targets is not None and w < 1:
        ok = (targets >= 0) & (targets < vocab)
        hit = wide.clone().scatter_(1, targets.long().masked_fill(~ok, vocab).unsqueeze(-1), 1.0)[:, :vocab]
        s = s + (1 - w) * (q1 * ok.double().unsqueeze(-1) + hit)
    return s * (1 - torch.tanh(x / cap) ** 2) / x.shape[0]


def rms(v, eps):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps)


def sandwich(x, y, post, pre, eps, gate, alpha):
    """float64 (x' before its rounding, the size of its summands)."""
    n = (1.0 if gate is None else gate) * (rms(y, eps) * post)
    return alpha * x + n, (alpha * x).abs() + n.abs()


def sandwich_bwd(x_new, y, post, pre, eps, gate, alpha, g, gh):
    """The gradients by their formulas in float64, from x' as it was kept: {name: (value, size of its summands)}."""
    gate_ = 1.0 if gate is None else gate
    r = 1 / torch.sqrt((x_new * x_new).mean(-1, keepdim=True) + eps)
    s = 1 / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    xh, yh = x_new * r, y * s
    a = gh * pre
    d = g + r * (a - xh * (a * xh).mean(-1, keepdim=True))
    d_abs = g.abs() + r * (a.abs() + xh.abs() * (a * xh).abs().mean(-1, keepdim=True))
    t, t_abs = gate_ * post * d, (gate_ * post).abs() * d_abs if gate is not None else post.abs() * d_abs
    out = {"dx": (alpha * d, abs(alpha) * d_abs),
           "dbranch": (s * (t - yh * (t * yh).mean(-1, keepdim=True)), s * (t_abs + yh.abs() * (t_abs * yh.abs()).mean(-1, keepdim=True))),
           "dpost": ((gate_ * d * yh).sum(0), (torch.as_tensor(gate_).abs().to(d) * d_abs * yh.abs()).sum(0)),
           "dpre": ((gh * xh).sum(0), (gh * xh).abs().sum(0))}
    if gate is not None:
        v, v_abs = d * yh * post, d_abs * yh.abs() * post.abs()
        out["dgate"] = (v.sum(0), v_abs.sum(0)) if gate.dim() == 1 else (v.sum(-1, keepdim=True), v_abs.sum(-1, keepdim=True))
    return out

"""The operators of a distillation step, as cases that can be timed and compared.

  top       `losses.top_logits`: a teacher's top logits, their log-probabilities and the log-mass of all others
  distill   `losses.capped_distillation`: a student's loss against those, forward and backward, or the loss alone
  norm      `kernels.sandwich_norm`: the norm behind a block, its gate, the residual add and the norm before the next
            block, forward and backward, or forward with the quantised output in front of an FP8 linear

`own` False: each in elementary float32 operations; True: the framework's calls.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5


# ---- the cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # a teacher looks at one token: the smallest call, all latency
        dict(name="top_1x50257_k64", op="top", rows=1, vocab=50257, k=64, cap=15.0, temp=1.0),
        # the teacher of the small model, eight sequences of 128 tokens over a vocabulary of bytes
        dict(name="top_1024x256_k8", op="top", rows=1024, vocab=256, k=8, cap=15.0, temp=2.0),
        # eight sequences of 1024 tokens at the pre-training vocabulary, many logits kept
        dict(name="top_8192x50304_k256", op="top", rows=8192, vocab=50304, k=256, cap=15.0, temp=2.0),
        # a step of the small model: one sequence of 128 tokens, all launches
        dict(name="distill_128x256_k8", op="distill", rows=128, vocab=256, k=8, cap=15.0, temp=2.0, weight=0.5, rest=True,
             padded=False, grad=True),
        # eight sequences of 1024 tokens with hard targets beside the teacher's, a vocabulary that is no multiple of 8
        dict(name="distill_8192x50257_k64", op="distill", rows=8192, vocab=50257, k=64, cap=15.0, temp=2.0, weight=0.5, rest=True,
             padded=False, grad=True),
        # the teacher alone at temperature one, a padded batch, the teacher's probabilities made to sum to one over the kept logits
        dict(name="distill_4096x50304_k32", op="distill", rows=4096, vocab=50304, k=32, cap=30.0, temp=1.0, weight=1.0, rest=False,
             padded=True, grad=True),
        # evaluation on a ragged batch: the loss alone
        dict(name="distill_1501x50257_k128_eval", op="distill", rows=1501, vocab=50257, k=128, cap=15.0, temp=1.0, weight=0.9, rest=True,
             padded=True, grad=False),
        # a junction of the small model
        dict(name="norm_128x128", op="norm", rows=128, cols=128, gate="channel", residual=1.0, quant=False, train=True),
        # the norm benchmark configuration
        dict(name="norm_32768x2048_channel", op="norm", rows=32768, cols=2048, gate="channel", residual=0.9, quant=False, train=True),
        # a ragged batch of wide rows, a gate per token
        dict(name="norm_3001x4096_token", op="norm", rows=3001, cols=4096, gate="token", residual=1.0, quant=False, train=True),
        # the pre-training model's junction without a gate: 16 sequences of 1024 tokens
        dict(name="norm_16384x1024", op="norm", rows=16384, cols=1024, gate="none", residual=1.0, quant=False, train=True),
        # a decode batch in front of an FP8 linear of a wide model (the values that the bytes stand for come back)
        dict(name="norm_16x8192_quant", op="norm", rows=16, cols=8192, gate="channel", residual=1.0, quant=True, train=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("top", "distill", "distill", "norm", "norm"))
    if op in ("top", "distill"):
        vocab = _log(rng, 256, 65536)
        if rng.random() < 0.4:
            vocab = max(256, vocab // 64 * 64)          # vocabularies are often padded
        rows = min(_log(rng, 1, 16384), 400_000_000 // vocab)
        k = min(_log(rng, 1, 256), vocab // 4)
        case = dict(op=op, rows=rows, vocab=vocab, k=k, cap=rng.choice((15.0, 30.0)), temp=rng.choice((1.0, 2.0, 4.0)))
        if op == "distill":
            case.update(weight=rng.choice((0.5, 0.9, 1.0)), rest=rng.random() < 0.7, padded=rng.random() < 0.3, grad=rng.random() < 0.8)
        return case
    quant = rng.random() < 0.3
    cols = 128 * _log(rng, 1, 64) if quant else 8 * _log(rng, 16, 1024)
    return dict(op="norm", rows=min(_log(rng, 1, 32768), 67_000_000 // cols), cols=cols, gate=rng.choice(("none", "channel", "token")),
                residual=rng.choice((1.0, 0.9, 0.5)), quant=quant, train=not quant and rng.random() < 0.8)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _logits(gen, rows, vocab):
    """An unembedding's output: most logits small, eight of a row well above the others, some of those beyond the cap."""
    x = torch.randn((rows, vocab), device="cuda", generator=gen).mul_(2.0)
    top = torch.randint(0, vocab, (rows, 8), device="cuda", generator=gen)
    x.scatter_(1, top, 4 + 14 * torch.rand((rows, 8), device="cuda", generator=gen))
    return x


def _activations(gen, shape):
    """N(0, 1) with one value in a thousand thirty times as large, as outlier features are."""
    x = torch.randn(shape, device="cuda", generator=gen)
    return torch.where(torch.rand(shape, device="cuda", generator=gen) < 1e-3, 30 * x, x).to(torch.bfloat16)


def _around_one(gen, n):
    return (1 + 0.1 * torch.randn(n, device="cuda", generator=gen)).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "norm":
        rows, cols, train = case["rows"], case["cols"], case["train"]
        shape = (rows, cols)
        gate = {"none": lambda: None, "channel": lambda: (0.5 * torch.randn(cols, device="cuda", generator=gen)).to(torch.bfloat16),
                "token": lambda: torch.rand((rows, 1), device="cuda", generator=gen).to(torch.bfloat16)}[case["gate"]]()
        state = dict(case, x=_activations(gen, shape), branch=_activations(gen, shape), post=_around_one(gen, cols), pre=_around_one(gen, cols),
                     gate_values=gate, g_new=torch.randn(shape, device="cuda", generator=gen).to(torch.bfloat16),
                     g_h=torch.randn(shape, device="cuda", generator=gen).to(torch.bfloat16))
        state["leaves"] = [t for t in (state["x"], state["branch"], state["post"], state["pre"], gate) if t is not None]
        if train:
            for t in state["leaves"]:
                t.requires_grad_()
        return state
    rows, vocab, k = case["rows"], case["vocab"], case["k"]
    x = _logits(gen, rows, vocab)
    state = dict(case, logits=x.to(torch.bfloat16))
    if case["op"] == "top":
        return state
    # a teacher that agrees with the student on some of it
    z = x.mul_(0.8).add_(torch.randn((rows, vocab), device="cuda", generator=gen)).div_(case["cap"]).tanh_().mul_(case["cap"] / case["temp"])
    z, ids = torch.topk(z.sub_(torch.logsumexp(z, -1, keepdim=True)), k)
    log_rest = torch.log1p(-z.exp().sum(-1).clamp_max(1 - 1e-6))
    if not case["rest"]:
        z, log_rest = torch.log_softmax(z, -1), None
    targets = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.5, ids[:, 0],
                          torch.randint(0, vocab, (rows,), device="cuda", generator=gen))
    if case["padded"]:                                   # the last eighth of the batch is padding; some entries of other rows are missing
        ids[rows - rows // 8:] = -1
        ids[:rows // 4, k // 2:k // 2 + 1] = -1
        targets[rows - rows // 8:] = -1
        if log_rest is not None:
            log_rest[rows - rows // 8:] = 0.0
    state.update(ids=ids.to(torch.int32), logp=z.contiguous(), log_rest=log_rest, targets=targets if case["weight"] < 1 else None)
    if case["grad"]:
        state["logits"].requires_grad_()
    return state


# ---- one pass --------------------------------------------------------------------------------------------------

def _plain_top(s):
    x = s["logits"]
    bits = x.view(torch.int16).to(torch.int64)
    order = torch.where(bits < 0, -(bits & 0x7fff), bits) * 2 ** 32 - torch.arange(x.shape[1], device=x.device)    # ties: the lowest index
    ids = order.topk(s["k"], -1).indices
    z = s["cap"] / s["temp"] * torch.tanh(x.float() / s["cap"])
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    kept, rest = e.gather(1, ids).sum(-1), e.scatter(1, ids, 0.0).sum(-1)
    total = kept + rest
    log_rest = torch.where(kept < rest, torch.log1p(-kept / total), torch.log(rest / total))     # near 0: from the smaller part
    return {"ids": ids.to(torch.int32), "logp": z.gather(1, ids) - (m + torch.log(total).unsqueeze(-1)), "log_rest": log_rest}


def _plain_distill(s):
    x, c, t, w = s["logits"].detach().float(), s["cap"], s["temp"], s["weight"]
    rows, vocab = x.shape
    ids = s["ids"].long()
    there = (ids >= 0) & (ids < vocab)
    at = torch.where(there, ids, 0)
    p = torch.where(there, torch.exp(s["logp"]), 0.0)
    rest = s["log_rest"] if s["log_rest"] is not None else torch.full((rows,), -math.inf, device=x.device)
    p_rest = torch.exp(rest)
    th = torch.tanh(x / c)
    z = c * th
    m = z.amax(-1, keepdim=True)
    e = torch.exp((z - m) / t)
    kept = torch.zeros_like(x).scatter_add_(1, at, there.float()) > 0
    tail, top = torch.where(kept, 0.0, e).sum(-1), torch.where(kept, e, 0.0).sum(-1)
    total = (top + tail).unsqueeze(-1)
    log_total = torch.log(total)
    log_tail = torch.where(top < tail, torch.log1p(-top / (top + tail)), torch.log(tail / (top + tail)))     # near 0: from the smaller part
    log_q = (z.gather(1, at) - m) / t - log_total
    row = w * t * t * (torch.where(p > 0, p * (s["logp"] - log_q), 0.0).sum(-1)
                       + torch.where(p_rest > 0, p_rest * (rest - log_tail), 0.0))
    if s["targets"] is not None:
        has = (s["targets"] >= 0) & (s["targets"] < vocab)
        target = torch.where(has, s["targets"], 0).unsqueeze(-1)
        e1 = torch.exp(z - m)
        total1 = e1.sum(-1, keepdim=True)
        row = row + torch.where(has, (1 - w) * (torch.log(total1) + m - z.gather(1, target)).squeeze(-1), 0.0)
    loss = row.mean()
    if not s["grad"]:
        return {"loss": loss}
    mass = (p.sum(-1) + p_rest).unsqueeze(-1)
    off = torch.where(p_rest > 0, p_rest / tail, 0.0).unsqueeze(-1)          # p_R / q_R, over the sum
    d = w * t * (e / total * mass - torch.where(kept, 0.0, e * off) - torch.zeros_like(x).scatter_add_(1, at, p))
    if s["targets"] is not None:
        hard = (1 - w) * has.float().unsqueeze(-1)
        d = d + hard * (e1 / total1) - torch.zeros_like(x).scatter_add_(1, target, hard)
    return {"loss": loss, "dlogits": (d * (1 - th * th) / rows).to(torch.bfloat16)}


def _plain_norm(s):
    x, y, post, pre = (s[n].detach().float() for n in ("x", "branch", "post", "pre"))
    gate = 1.0 if s["gate_values"] is None else s["gate_values"].detach().float()
    r_y = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    y_hat = y * r_y
    new = (s["residual"] * x + gate * (y_hat * post)).to(torch.bfloat16)     # the residual stream, as it is kept
    r = torch.rsqrt(new.float().square().mean(-1, keepdim=True) + EPS)
    x_hat = new.float() * r
    h = (x_hat * pre).to(torch.bfloat16)
    if s["quant"]:
        tiles = h.float().view(h.shape[0], -1, 128)
        scale = (tiles.abs().amax(-1, keepdim=True) / 448.0).clamp_min(1e-30)
        q = (tiles / scale).to(torch.float8_e4m3fn)
        return {"new": new, "h": (q.float() * scale).to(torch.bfloat16).view_as(h)}
    if not s["train"]:
        return {"new": new, "h": h}
    g_h = s["g_h"].float()
    a = g_h * pre
    d = s["g_new"].float() + r * (a - x_hat * (a * x_hat).mean(-1, keepdim=True))
    t = gate * post * d
    out = {"new": new, "h": h, "dx": s["residual"] * d, "dbranch": r_y * (t - y_hat * (t * y_hat).mean(-1, keepdim=True)),
           "dpost": (gate * d * y_hat).sum(0), "dpre": (g_h * x_hat).sum(0)}
    if s["gate_values"] is not None:
        dg = d * y_hat * post
        out["dgate"] = dg.sum(0) if s["gate"] == "channel" else dg.sum(-1, keepdim=True)
    return {n: v.to(torch.bfloat16) for n, v in out.items()}


def _own(s):
    from train_gpt_b200 import kernels, losses
    if s["op"] == "top":
        top = losses.top_logits(s["logits"], s["cap"], s["k"], temperature=s["temp"])
        return {"ids": top.ids, "logp": top.logp, "log_rest": top.log_rest}
    if s["op"] == "distill":
        x = s["logits"]
        x.grad = None
        loss = losses.capped_distillation(x, losses.TopLogits(s["ids"], s["logp"], s["log_rest"]), s["cap"], target_ids=s["targets"],
                                          temperature=s["temp"], weight=s["weight"])
        if not s["grad"]:
            return {"loss": loss}
        loss.backward()
        return {"loss": loss.detach(), "dlogits": x.grad}
    if s["quant"]:
        new, h = kernels.sandwich_norm_quant(s["x"], s["branch"], s["post"], s["pre"], EPS, gate=s["gate_values"], residual_scale=s["residual"])
        return {"new": new, "h": (h.q.view(new.shape[0], -1, 128).float() * h.scales.unsqueeze(-1)).to(torch.bfloat16).view_as(new)}
    new, h = kernels.sandwich_norm(s["x"], s["branch"], s["post"], s["pre"], EPS, gate=s["gate_values"], residual_scale=s["residual"])
    if not s["train"]:
        return {"new": new, "h": h}
    grads = torch.autograd.grad((new, h), s["leaves"], (s["g_new"], s["g_h"]))
    return {"new": new.detach(), "h": h.detach(), **dict(zip(("dx", "dbranch", "dpost", "dpre", "dgate"), grads))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"top": _plain_top, "distill": _plain_distill, "norm": _plain_norm}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    if case["op"] == "norm":
        e, train = case["rows"] * case["cols"], case["train"]
        # x and the branch's output in, the new stream and its norm out; in training two gradients in and two out
        per = 2 + 2 + 2 + (1 + 4 / 128 if case["quant"] else 2) + (8 if train else 0)
        vectors = 2 + (case["gate"] == "channel")
        return {"bytes": per * e + 2.0 * vectors * case["cols"] * (2 if train else 1), "flops": (40.0 if train else 12.0) * e}
    rows, e = case["rows"], case["rows"] * case["vocab"]
    if case["op"] == "top":
        return {"bytes": 2.0 * e + rows * (8.0 * case["k"] + 4), "flops": 8.0 * e}
    given = rows * (8.0 * case["k"] + (4 if case["rest"] else 0) + (8 if case["weight"] < 1 else 0))
    both = case["weight"] < 1 and case["temp"] != 1
    return {"bytes": (4.0 if case["grad"] else 2.0) * e + given, "flops": ((20.0 if both else 16.0) if case["grad"] else (10.0 if both else 8.0)) * e}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _exact_top(s, lo, hi):
    x = s["logits"][lo:hi].double()
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :s["k"]]
    logq = torch.log_softmax(s["cap"] * torch.tanh(x / s["cap"]) / s["temp"], -1)
    return {"ids": ids.to(torch.int32), "logp": logq.gather(1, ids), "log_rest": logq.scatter(1, ids, -math.inf).logsumexp(-1)}


def _exact_distill(s, lo, hi):
    """The rows' share of the loss, and its gradient by differentiation."""
    x = s["logits"].detach()[lo:hi].double().requires_grad_()
    vocab, t, w = x.shape[1], s["temp"], s["weight"]
    with torch.enable_grad():
        z = s["cap"] * torch.tanh(x / s["cap"])
        logq = torch.log_softmax(z / t, -1)
        ids, logp = s["ids"][lo:hi].long(), s["logp"][lo:hi].double()
        there = (ids >= 0) & (ids < vocab)
        logp = logp.masked_fill(~there, -math.inf)
        took = torch.zeros((x.shape[0], vocab + 1), device=x.device, dtype=torch.bool).scatter_(1, ids.masked_fill(~there, vocab), True)[:, :vocab]
        seen = logq.gather(1, ids.masked_fill(~there, 0))
        loss = w * t ** 2 * (logp.exp() * (logp.masked_fill(~there, 0.0) - seen)).sum()
        if s["log_rest"] is not None:
            rest = s["log_rest"][lo:hi].double()
            loss = loss + w * t ** 2 * (rest.exp() * (rest - logq.masked_fill(took, -math.inf).logsumexp(-1))).sum()
        if s["targets"] is not None:
            targets = s["targets"][lo:hi].long()
            has = (targets >= 0) & (targets < vocab)
            loss = loss - (1 - w) * (torch.log_softmax(z, -1).gather(1, targets.masked_fill(~has, 0).unsqueeze(-1)).squeeze(-1) * has).sum()
        loss = loss / s["rows"]
        d = torch.autograd.grad(loss, x)[0] if s["grad"] else None
    return {"loss": loss.detach(), "dlogits": d}


def _rms(v):
    return v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)


def _exact_norm(s, lo, hi):
    """The junction by its definition, and its gradients by differentiation; those of the vectors are these rows' share."""
    leaves = [s[n].detach() for n in ("x", "branch", "post", "pre")] + ([] if s["gate_values"] is None else [s["gate_values"].detach()])
    leaves = [(v[lo:hi] if v.dim() == 2 else v).double().requires_grad_() for v in leaves]
    x, y, post, pre = leaves[:4]
    with torch.enable_grad():
        new = s["residual"] * x + (leaves[4] if len(leaves) == 5 else 1.0) * (_rms(y) * post)
        new = new + (new.to(torch.bfloat16).double() - new).detach()         # kept in bf16; the rounding passes gradients through
        h = _rms(new) * pre
        if s["train"]:
            grads = torch.autograd.grad((new, h), leaves, (s["g_new"][lo:hi].double(), s["g_h"][lo:hi].double()))
            return {"new": new.detach(), "h": h.detach(), **dict(zip(("dx", "dbranch", "dpost", "dpre", "dgate"), grads))}
    h = h.detach()
    if s["quant"]:
        tiles = h.to(torch.bfloat16).double().view(h.shape[0], -1, 128)
        scale = (tiles.abs().amax(-1, keepdim=True) / 448).clamp_min(1e-30)
        h = ((tiles / scale).float().to(torch.float8_e4m3fn).double() * scale).view_as(h)
    return {"new": new.detach(), "h": h}


def exact(case, seed):
    s = prepare(case, seed)
    part = {"top": _exact_top, "distill": _exact_distill, "norm": _exact_norm}[case["op"]]
    rows = case["rows"]
    step = max(1, 2 ** 25 // case["cols" if case["op"] == "norm" else "vocab"])
    parts = [part(s, lo, min(rows, lo + step)) for lo in range(0, rows, step)]
    out = {}
    for n in parts[0]:
        values = [p[n] for p in parts]
        if values[0] is not None:
            out[n] = torch.cat(values) if values[0].dim() > 1 or n == "log_rest" else torch.stack(values).sum(0)
    return out

"""The operators of a block with rotary positions, a gated feed-forward and residual dropout, as cases that can be timed and compared.

  qk      `kernels.qk_norm_rope`: the norm of every head of queries and keys and the rotation by position, forward and backward
  ffn     `kernels.gated_linear`: act(x w_gate) * (x w_up), forward and backward
  drop    `kernels.dropout`: dropout of a branch and its add to the residual stream, forward and backward

`own` False: each in elementary float32 operations; True: the framework's calls.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

EPS = 1e-5


# ---- the cases -------------------------------------------------------------------------------------------------

def listed():
    return [
        # one new token of each of sixteen sequences that are far into a long context: all latency
        dict(name="qk_16x1_h32k8_d128", op="qk", batch=16, tokens=1, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=True,
             packed=False, far=131072, theta=500000.0, train=False),
        # the pre-training model's attention: 32 sequences of 1024 tokens, 16 heads of 64, out of one projection
        dict(name="qk_32x1024_h16k16_d64", op="qk", batch=32, tokens=1024, heads=16, kv_heads=16, dim=64, rotary=64, interleaved=False, norm=True,
             packed=True, far=0, theta=10000.0, train=True),
        # a ragged batch of a model that rotates a part of each head, in neighbouring pairs
        dict(name="qk_3x1021_h12k4_d80_part", op="qk", batch=3, tokens=1021, heads=12, kv_heads=4, dim=80, rotary=32, interleaved=True, norm=True,
             packed=True, far=4096, theta=10000.0, train=True),
        # one long sequence of a wide model, grouped keys, its heads rotated and not normed
        dict(name="qk_1x32768_h32k8_d128_rope", op="qk", batch=1, tokens=32768, heads=32, kv_heads=8, dim=128, rotary=128, interleaved=False, norm=False,
             packed=True, far=0, theta=500000.0, train=True),
        # one token through the pre-training model's feed-forward: the weights are read once
        dict(name="ffn_1x1024x4096", op="ffn", rows=1, cols=1024, inner=4096, act="silu", train=False),
        # a decode batch of a wide model
        dict(name="ffn_16x8192x8192", op="ffn", rows=16, cols=8192, inner=8192, act="silu", train=False),
        # a step of the small model: one sequence of 128 tokens, all launches
        dict(name="ffn_128x128x512_train", op="ffn", rows=128, cols=128, inner=512, act="gelu", train=True),
        # a ragged batch, an inner width that no tile divides
        dict(name="ffn_1501x2048x5464_train", op="ffn", rows=1501, cols=2048, inner=5464, act="silu", train=True),
        # the pre-training step: 32 sequences of 1024 tokens
        dict(name="ffn_32768x1024x4096_train", op="ffn", rows=32768, cols=1024, inner=4096, act="silu", train=True),
        # a branch of the small model
        dict(name="drop_128x128", op="drop", rows=128, cols=128, p=0.1, residual=True, train=True),
        # the pre-training step's branch
        dict(name="drop_32768x1024", op="drop", rows=32768, cols=1024, p=0.1, residual=True, train=True),
        # a ragged batch of a wide model, without a residual stream
        dict(name="drop_4093x8191", op="drop", rows=4093, cols=8191, p=0.5, residual=False, train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("qk", "ffn", "ffn", "drop"))
    if op == "qk":
        dim = rng.choice((32, 48, 64, 80, 96, 128, 128, 192, 256))
        kv_heads = _log(rng, 1, 16)
        heads = kv_heads * rng.choice((1, 1, 2, 4))
        batch = _log(rng, 1, 64)
        per_token = (heads + kv_heads) * dim
        tokens = max(1, min(_log(rng, 1, 32768), 100_000_000 // (batch * per_token)))
        rotary = dim if rng.random() < 0.7 else 16 * rng.randint(1, dim // 16)
        return dict(op="qk", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, interleaved=rng.random() < 0.3,
                    norm=rng.random() < 0.8, packed=rng.random() < 0.6, far=rng.choice((0, 4096, 131072, 1000000)),
                    theta=rng.choice((10000.0, 500000.0)), train=rng.random() < 0.7)
    if op == "ffn":
        cols, inner = 8 * _log(rng, 8, 1024), 8 * _log(rng, 8, 1024)
        if rng.random() < 0.5:
            cols, inner = max(64, cols // 64 * 64), max(64, inner // 64 * 64)
        rows = max(1, min(_log(rng, 1, 32768), 120_000_000_000 // (cols * inner), 100_000_000 // max(cols, inner)))
        return dict(op="ffn", rows=rows, cols=cols, inner=inner, act=rng.choice(("silu", "gelu", "relu")), train=rng.random() < 0.6)
    cols = _log(rng, 64, 16384)
    return dict(op="drop", rows=min(_log(rng, 1, 32768), 33_000_000 // cols), cols=cols, p=rng.choice((0.05, 0.1, 0.2, 0.5)),
                residual=rng.random() < 0.6, train=rng.random() < 0.8)


# ---- inputs ----------------------------------------------------------------------------------------------------

def _normal(gen, *shape, std=1.0):
    return (std * torch.randn(shape, device="cuda", generator=gen)).to(torch.bfloat16)


def _activations(gen, *shape):
    """N(0, 1) with one value in a thousand twenty times as large, as outlier features are."""
    x = torch.randn(shape, device="cuda", generator=gen)
    return torch.where(torch.rand(shape, device="cuda", generator=gen) < 1e-3, 20 * x, x).to(torch.bfloat16)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    if case["op"] == "qk":
        b, t, h, kh, d = case["batch"], case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        if case["packed"]:                               # queries, keys and values side by side, as one projection leaves them
            qkv = _activations(gen, b, t, (h + 2 * kh) * d)
            q, k = qkv[..., :h * d].unflatten(-1, (h, d)), qkv[..., h * d:(h + kh) * d].unflatten(-1, (kh, d))
        else:
            q, k = _activations(gen, b, t, h, d), _activations(gen, b, t, kh, d)
        scales = [(1 + 0.2 * torch.randn(d, device="cuda", generator=gen)).to(torch.bfloat16) for _ in range(2)] if case["norm"] else [None, None]
        positions = None
        if case["far"]:                                  # every sequence begins somewhere
            positions = torch.randint(0, case["far"], (b, 1), device="cuda", generator=gen) + torch.arange(t, device="cuda")
        state.update(q=q, k=k, q_scale=scales[0], k_scale=scales[1], positions=positions)
        state["leaves"] = [v for v in (q, k, *scales) if v is not None]
        if case["train"]:
            state.update(g_q=_normal(gen, b, t, h, d), g_k=_normal(gen, b, t, kh, d))
    elif case["op"] == "ffn":
        m, n, f = case["rows"], case["cols"], case["inner"]
        state.update(x=_activations(gen, m, n), w_gate=_normal(gen, n, f, std=n ** -0.5), w_up=_normal(gen, n, f, std=n ** -0.5))
        state["leaves"] = [state["x"], state["w_gate"], state["w_up"]]
        if case["train"]:
            state["g"] = _normal(gen, m, f, std=m ** -0.5)
    else:
        shape = (case["rows"], case["cols"])
        state.update(x=_activations(gen, *shape), res=_activations(gen, *shape) if case["residual"] else None,
                     seed=torch.randint(-2 ** 62, 2 ** 62, (1,), device="cuda", generator=gen), site=int(seed) % 97)
        state["leaves"] = [v for v in (state["x"], state["res"]) if v is not None]
        if case["train"]:
            state["g"] = _normal(gen, *shape)
    if case["train"]:
        for v in state["leaves"]:
            v.requires_grad_()
    return state


# ---- one pass --------------------------------------------------------------------------------------------------

def _plain_angles(s, device):
    positions = s["positions"] if s["positions"] is not None else torch.arange(s["tokens"], device=device).expand(s["batch"], -1)
    rotary = s["rotary"]
    turn = s["theta"] ** (-torch.arange(0, rotary, 2, device=device, dtype=torch.float64) / rotary)
    angle = positions.double().unsqueeze(-1) * turn                          # in 64 bits: far positions have many turns behind them
    return torch.cos(angle).float().unsqueeze(-2), torch.sin(angle).float().unsqueeze(-2)


def _plain_rotate(x, cos, sin, s):
    rotary = s["rotary"]
    x, rest = x[..., :rotary], x[..., rotary:]
    if s["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)
    a, b = x[..., :rotary // 2], x[..., rotary // 2:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)


def _plain_heads(x, scale, g, cos, sin, s):
    """One of queries and keys: rotated, its gradient, its scale's gradient."""
    x = x.detach().float()
    if scale is None:
        y = _plain_rotate(x, cos, sin, s).to(torch.bfloat16)
        return (y,) if g is None else (y, _plain_rotate(g.float(), cos, -sin, s).to(torch.bfloat16), None)
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    x_hat, w = x * r, scale.detach().float()
    y = _plain_rotate(x_hat * w, cos, sin, s).to(torch.bfloat16)
    if g is None:
        return (y,)
    g = _plain_rotate(g.float(), cos, -sin, s)
    a = g * w
    dx = r * (a - x_hat * (a * x_hat).mean(-1, keepdim=True))
    return y, dx.to(torch.bfloat16), (g * x_hat).sum((0, 1, 2)).to(torch.bfloat16)


def _plain_qk(s):
    cos, sin = _plain_angles(s, s["q"].device)
    train = s["train"]
    q = _plain_heads(s["q"], s["q_scale"], s["g_q"] if train else None, cos, sin, s)
    k = _plain_heads(s["k"], s["k_scale"], s["g_k"] if train else None, cos, sin, s)
    out = {"q": q[0], "k": k[0]}
    if train:
        out.update(dq=q[1], dk=k[1])
        if s["norm"]:
            out.update(dq_scale=q[2], dk_scale=k[2])
    return out


def _plain_act(g, act):
    """(act(g), its derivative)"""
    if act == "relu":
        return g.clamp_min(0), (g > 0).float()
    if act == "silu":
        sig = torch.sigmoid(g)
        return g * sig, sig * (1 + g * (1 - sig))
    phi = 0.5 * torch.erfc(-g / math.sqrt(2))
    return g * phi, phi + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def _plain_ffn(s):
    x, wg, wu = (s[n].detach().float() for n in ("x", "w_gate", "w_up"))
    gate, up = x @ wg, x @ wu
    a, da = _plain_act(gate, s["act"])
    out = {"h": a * up}
    if s["train"]:
        g = s["g"].float()
        d_gate, d_up = g * up * da, g * a
        out.update(dx=d_gate @ wg.T + d_up @ wu.T, dw_gate=x.T @ d_gate, dw_up=x.T @ d_up)
    return {n: v.to(torch.bfloat16) for n, v in out.items()}


def _plain_random(seed, site, n):
    """16 random bits for each of n elements: Philox4x32 with ten rounds, the counter (piece of eight elements, site, 0), the key the seed."""
    m0, m1, low = 0xD2511F53, 0xCD9E8D57, 0xFFFFFFFF
    piece = torch.arange((n + 7) // 8, device=seed.device)
    c0, c1 = piece & low, piece >> 32
    c2, c3 = torch.full_like(piece, site), torch.zeros_like(piece)
    k0, k1 = seed & low, (seed >> 32) & low

    def round_(c0, c1, c2, c3, i):
        a, b = c0 * m0, c2 * m1                          # (64-bit products, of which the sign is a bit like any other)
        j0, j1 = (k0 + i * 0x9E3779B9) & low, (k1 + i * 0xBB67AE85) & low
        return ((b >> 32) & low) ^ c1 ^ j0, b & low, ((a >> 32) & low) ^ c3 ^ j1, a & low

    c = (c0, c1, c2, c3)
    c = round_(*round_(*round_(*round_(*round_(*c, 0), 1), 2), 3), 4)
    c = round_(*round_(*round_(*round_(*round_(*c, 5), 6), 7), 8), 9)
    words = torch.stack(c, -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).flatten()[:n]


def _plain_drop(s):
    x = s["x"].detach().float()
    threshold = round(s["p"] * 65536)
    keep = (_plain_random(s["seed"], s["site"], x.numel()) >= threshold).view_as(x)
    scale = 65536 / (65536 - threshold)
    y = torch.where(keep, x * scale, 0.0)
    if s["res"] is not None:
        y = y + s["res"].detach().float()
    out = {"y": y.to(torch.bfloat16)}
    if s["train"]:
        out["dx"] = torch.where(keep, s["g"].float() * scale, 0.0).to(torch.bfloat16)
        if s["res"] is not None:
            out["dres"] = s["g"]
    return out


def _own(s):
    from train_gpt_b200 import kernels
    train = s["train"]
    if s["op"] == "qk":
        q, k = kernels.qk_norm_rope(s["q"], s["k"], s["q_scale"], s["k_scale"], EPS, s["positions"], theta=s["theta"], rotary_dim=s["rotary"],
                                    interleaved=s["interleaved"])
        out = {"q": q.detach(), "k": k.detach()}
        if train:
            out.update(zip(("dq", "dk", "dq_scale", "dk_scale"), torch.autograd.grad((q, k), s["leaves"], (s["g_q"], s["g_k"]))))
        return out
    if s["op"] == "ffn":
        h = kernels.gated_linear(s["x"], s["w_gate"], s["w_up"], s["act"])
        out = {"h": h.detach()}
        if train:
            out.update(zip(("dx", "dw_gate", "dw_up"), torch.autograd.grad(h, s["leaves"], s["g"])))
        return out
    y = kernels.dropout(s["x"], s["p"], s["seed"], site=s["site"], residual=s["res"])
    out = {"y": y.detach()}
    if train:
        out.update(zip(("dx", "dres"), torch.autograd.grad(y, s["leaves"], s["g"])))
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"qk": _plain_qk, "ffn": _plain_ffn, "drop": _plain_drop}[state["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------

def work(case):
    train = case["train"]
    if case["op"] == "qk":
        tokens = case["batch"] * case["tokens"]
        e = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        # in and out; backward the gradient in and out, and with a norm its input again
        per = 4 + ((6 if case["norm"] else 4) if train else 0)
        return {"bytes": float(per * e + (8 * tokens if case["far"] else 0) + (4 * case["dim"] if case["norm"] else 0)),
                "flops": float(e * (8 + (16 if train else 0)))}
    if case["op"] == "ffn":
        m, n, f = case["rows"], case["cols"], case["inner"]
        # x, both weights, h; backward the gradient of h, x and the weights again, and their gradients
        return {"bytes": 2.0 * (m * n + 2 * n * f + m * f) + (2.0 * (m * f + 2 * m * n + 4 * n * f) if train else 0.0),
                "flops": 4.0 * m * n * f * (3 if train else 1)}
    e = case["rows"] * case["cols"]
    return {"bytes": float((4 + (2 if case["residual"] else 0) + (4 if train else 0)) * e), "flops": float((20 if train else 10) * e)}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------

def _exact_qk(s):
    """Each head as complex numbers of which a turn is a product; gradients by differentiation."""
    leaves = [v.detach().double().requires_grad_() for v in s["leaves"]]
    rotary, positions = s["rotary"], s["positions"]
    if positions is None:
        positions = torch.arange(s["tokens"], device="cuda").repeat(s["batch"], 1)
    i = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), positions.double()[..., None, None] / torch.pow(s["theta"], 2 * i / rotary))

    def heads(x, w):
        if w is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        part = x[..., :rotary]
        pairs = part.unflatten(-1, (rotary // 2, 2)) if s["interleaved"] else part.unflatten(-1, (2, rotary // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        return torch.cat(((z if s["interleaved"] else z.transpose(-1, -2)).flatten(-2), x[..., rotary:]), -1)

    with torch.enable_grad():
        q, k = heads(leaves[0], leaves[2] if s["norm"] else None), heads(leaves[1], leaves[3] if s["norm"] else None)
        out = {"q": q.detach(), "k": k.detach()}
        if s["train"]:
            out.update(zip(("dq", "dk", "dq_scale", "dk_scale"), torch.autograd.grad((q, k), leaves, (s["g_q"].double(), s["g_k"].double()))))
    return out


def _exact_ffn(s):
    """A range of rows at a time; gradients by differentiation, the weights' added up."""
    w = [s[n].detach().double().requires_grad_() for n in ("w_gate", "w_up")]
    act = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "relu": torch.relu}[s["act"]]
    parts, sums = [], None
    for lo in range(0, s["rows"], 8192):
        x = s["x"][lo:lo + 8192].detach().double().requires_grad_()
        with torch.enable_grad():
            h = act(x @ w[0]) * (x @ w[1])
            if not s["train"]:
                parts.append({"h": h.detach()})
                continue
            dx, *dw = torch.autograd.grad(h, (x, *w), s["g"][lo:lo + 8192].double())
        parts.append({"h": h.detach(), "dx": dx})
        sums = dw if sums is None else [a + b for a, b in zip(sums, dw)]
    out = {n: torch.cat([p[n] for p in parts]) for n in parts[0]}
    if sums is not None:
        out.update(dw_gate=sums[0], dw_up=sums[1])
    return out


def _exact_drop(s):
    n, cols = s["x"].numel(), s["cols"]
    key = int(s["seed"]) % 2 ** 64
    counter = np.arange((n + 7) // 8, dtype=np.uint64)
    low, half = np.uint64(2 ** 32 - 1), np.uint64(32)
    words = [counter & low, counter >> half, np.full_like(counter, s["site"]), np.zeros_like(counter)]
    keys = [key % 2 ** 32, key // 2 ** 32]
    for _ in range(10):
        p, q = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
        words = [(q >> half) ^ words[1] ^ np.uint64(keys[0]), q & low, (p >> half) ^ words[3] ^ np.uint64(keys[1]), p & low]
        keys = [(keys[0] + 0x9E3779B9) % 2 ** 32, (keys[1] + 0xBB67AE85) % 2 ** 32]
    bits = np.stack(words, 1).astype(np.uint32).view(np.uint16).reshape(-1)[:n].astype(np.int32)
    dropped = round(s["p"] * 65536)
    mask = torch.from_numpy(bits >= dropped).to("cuda").view(-1, cols).double() / (1 - dropped / 65536)
    out = {"y": s["x"].detach().double() * mask + (0 if s["res"] is None else s["res"].detach().double())}
    if s["train"]:
        out["dx"] = s["g"].double() * mask
        if s["res"] is not None:
            out["dres"] = s["g"].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"qk": _exact_qk, "ffn": _exact_ffn, "drop": _exact_drop}[case["op"]](s)

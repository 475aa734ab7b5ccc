"""Rows whose elements lie beyond 2^31 elements and 2^32 bytes of their tensor's start, for each distillation operator and the sandwich norm: the
same bits as those rows alone; and the junction written over its inputs, as the C entry allows."""
import pytest
import torch

pytestmark = pytest.mark.gpu
EPS = 1e-5


def _room(gib):
    if torch.cuda.mem_get_info()[0] < gib * 2 ** 30:
        pytest.skip(f"needs {gib} GB")


def _tail(rows, vocab, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(torch.bfloat16)


def test_logits():
    """65536 x 50257: the last 256 rows (a multiple of eight before them, so that they lie as in a tensor of their own; a power of two of the
    batch, so that the mean's factor only shifts the gradient)."""
    from train_gpt_b200 import losses, ops
    _room(30)
    rows, vocab, few = 65536, 50257, 256
    tail = _tail(few, vocab, 1)
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    x[-few:] = tail
    top = losses.top_logits(x, 15.0, 64, temperature=2.0)
    want = losses.top_logits(tail, 15.0, 64, temperature=2.0)
    assert torch.equal(top.ids[-few:], want.ids)
    # (how many rows an SM works on at once, and with that a sum's order, goes by the number of rows)
    assert float((top.logp[-few:] - want.logp).abs().max()) <= 2.0 ** -16 and float((top.log_rest[-few:] - want.log_rest).abs().max()) <= 2.0 ** -16
    top = losses.TopLogits(*(t.clone() for t in top))
    top.ids[-few:], top.logp[-few:], top.log_rest[-few:] = want
    for grad in (True, False):
        loss, d = ops.softcap_distill(x, *top, 15.0, None, 2.0, 1.0, want_grad=grad)
        loss_few, d_few = ops.softcap_distill(tail, *want, 15.0, None, 2.0, 1.0, want_grad=grad)
        # the sums of exp(z / T) and their logarithms, in another order: T^2 = 4 times 2^-17
        assert float((loss[-few:] - loss_few).abs().max()) <= 2.0 ** -15
        if grad:
            assert torch.equal(d[-few:], (d_few.float() / (rows // few)).to(torch.bfloat16))
            first = d[:1]
            assert torch.equal(d[1000:1001], first) and torch.equal(d[rows - few - 8:rows - few - 7], first)        # (a multiple of eight: of one alignment)
            del d, d_few


@pytest.mark.parametrize("gate", ["none", "channel", "token"])
def test_junction(gate):
    """280000 x 8192, the rows at its end against themselves alone, forward, quantised and backward."""
    from train_gpt_b200 import ops
    _room(40)
    rows, cols, few = 280000, 8192, 100
    g = torch.Generator(device="cuda").manual_seed(2)
    vectors = [(1 + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2)]
    parts = [_tail(few, cols, s) for s in range(4)]
    full = []
    for p in parts:
        t = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
        t[-few:] = p
        full.append(t)
    kinds = {"none": (None, None), "channel": (vectors[1], vectors[1]), "token": (torch.ones(rows, 1, dtype=torch.bfloat16, device="cuda"), torch.full((few, 1), 0.5, dtype=torch.bfloat16, device="cuda"))}
    gate_full, gate_few = kinds[gate]
    if gate == "token":
        gate_full[-few:] = 0.5
    a = ops.sandwich_norm_fwd(full[0], full[1], *vectors, EPS, gate=gate_full, residual_scale=0.9, want_q=True)
    b = ops.sandwich_norm_fwd(parts[0], parts[1], *vectors, EPS, gate=gate_few, residual_scale=0.9, want_q=True)
    for u, v in zip(a, b):
        u = u[-few:]
        assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))
    del a
    x_new = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    x_new[-few:] = b[0]
    da = ops.sandwich_norm_bwd(x_new, full[1], *vectors, EPS, full[2], full[3], gate=gate_full, residual_scale=0.9)
    db = ops.sandwich_norm_bwd(b[0], parts[1], *vectors, EPS, parts[2], parts[3], gate=gate_few, residual_scale=0.9)
    for i in (0, 1, 4) if gate == "token" else (0, 1):
        assert torch.equal(da[i][-few:], db[i])
    assert not da[0][:-few].any() and not da[1][:-few].any()


@pytest.mark.parametrize("rows,cols", [(5, 8), (700, 520), (2000, 2048), (300, 4616), (3000, 8192)])
@pytest.mark.parametrize("over", ["x", "branch"])
def test_the_junction_over_its_input(rows, cols, over):
    from train_gpt_b200 import _lib, ops
    x, y = _tail(rows, cols, 3), _tail(rows, cols, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    post, pre = ((1 + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(torch.bfloat16) for _ in range(2))
    gate = torch.rand(rows, 1, device="cuda", generator=g).to(torch.bfloat16)
    want = ops.sandwich_norm_fwd(x, y, post, pre, EPS, gate=gate, residual_scale=0.9)
    h, out = torch.empty_like(x), x if over == "x" else y
    assert _lib.load().tg_sandwich_norm_fwd(x.data_ptr(), y.data_ptr(), post.data_ptr(), pre.data_ptr(), gate.data_ptr(), 2, 0.9, EPS, out.data_ptr(), h.data_ptr(),
                                            None, None, rows, cols, torch.cuda.current_stream().cuda_stream) == _lib.TG_OK
    assert torch.equal(out, want[0]) and torch.equal(h, want[1])

"""What the distillation operators and the sandwich norm refuse, checked where it is refused: on the host, before any device work."""
import ctypes

import pytest
import torch

BF = torch.bfloat16


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


@pytest.fixture(scope="module")
def lib():
    from train_gpt_b200 import _lib, build
    build.build()
    return _lib.load()


def _sandwich(x=None, branch=None, post=None, pre=None, gate=None, **kw):
    from train_gpt_b200 import kernels
    x = _z(4, 128) if x is None else x
    d = x.shape[-1] if x.dim() else 8
    return kernels.sandwich_norm(x, _z(4, 128) if branch is None else branch, _z(d) if post is None else post, _z(d) if pre is None else pre, 1e-5, gate=gate, **kw)


@pytest.mark.parametrize("args,message", [
    (dict(x=_z(4, 64)), "branch shape"),
    (dict(post=_z(64)), "scale shape"),
    (dict(pre=_z(1, 128)), "scale shape"),
    (dict(gate=_z(64)), "gate shape"),
    (dict(gate=_z(4)), "gate shape"),
    (dict(gate=_z(1, 128)), "gate shape"),
    (dict(x=_z(4, 100), branch=_z(4, 100)), "multiple of 8"),
    (dict(x=_z(4, 8200), branch=_z(4, 8200)), "at most 8192"),
    (dict(x=_z(4, 0), branch=_z(4, 0)), "multiple of 8"),
    (dict(x=_z(), branch=_z()), "at least one dimension"),
])
def test_sandwich_shapes(args, message):
    with pytest.raises(ValueError, match=message):
        _sandwich(**args)


def test_no_cpu_path():
    from train_gpt_b200 import losses
    with pytest.raises(RuntimeError, match="no CPU path"):
        _sandwich()
    with pytest.raises(RuntimeError, match="no CPU path"):
        losses.top_logits(_z(2, 16), 15.0, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        losses.capped_distillation(_z(2, 16), losses.TopLogits(_z(2, 4, dtype=torch.int32), _z(2, 4, dtype=torch.float32)), 15.0)


@pytest.mark.parametrize("shape,cap,k,t,message", [
    ((2, 16), 15.0, 0, 1.0, "k=0"), ((2, 16), 15.0, 17, 1.0, "k=17"), ((2, 400), 15.0, 257, 1.0, "at most 256"), ((2, 2 ** 20 + 1), 15.0, 4, 1.0, "vocabulary of"),
    ((2, 0), 15.0, 1, 1.0, "no vocabulary"), ((), 15.0, 1, 1.0, "at least one dimension"), ((2, 16), 0.0, 4, 1.0, "cap="), ((2, 16), 65.0, 4, 1.0, "cap="),
    ((2, 16), float("nan"), 4, 1.0, "cap="), ((2, 16), 15.0, 4, 0.0, "temperature="), ((2, 16), 15.0, 4, -1.0, "temperature="), ((2, 16), 15.0, 4, 0.2, "temperature="),
    ((2, 16), 15.0, 4, 2000.0, "temperature="), ((2, 16), 15.0, 4, float("nan"), "temperature="),
])
def test_top_logits(shape, cap, k, t, message):
    from train_gpt_b200 import losses
    with pytest.raises(ValueError, match=message):
        losses.top_logits(_z(*shape), cap, k, temperature=t)


@pytest.mark.parametrize("change,message", [
    (dict(ids=_z(3, 4, dtype=torch.int32)), "teacher ids"), (dict(ids=_z(4, dtype=torch.int32)), "teacher ids"), (dict(logp=_z(2, 5, dtype=torch.float32)), "teacher logp"),
    (dict(rest=_z(2, 1, dtype=torch.float32)), "log_rest"), (dict(target_ids=_z(3, dtype=torch.int64), weight=0.5), "target_ids"), (dict(weight=0.5), "needs target_ids"),
    (dict(weight=-0.1), "weight="), (dict(weight=1.1), "weight="), (dict(weight=float("nan")), "weight="), (dict(temperature=0.1), "temperature="), (dict(cap=100.0), "cap="),
    (dict(logits=_z(2, 300), ids=_z(2, 257, dtype=torch.int32), logp=_z(2, 257, dtype=torch.float32)), "at most 256"),
])
def test_distillation(change, message):
    from train_gpt_b200 import losses
    a = dict(logits=_z(2, 16), ids=_z(2, 4, dtype=torch.int32), logp=_z(2, 4, dtype=torch.float32), rest=None, cap=15.0)
    a.update(change)
    teacher = losses.TopLogits(a.pop("ids"), a.pop("logp"), a.pop("rest"))
    with pytest.raises(ValueError, match=message):
        losses.capped_distillation(a.pop("logits"), teacher, a.pop("cap"), **a)


def test_c_entries(lib):
    """(aligned numbers stand for addresses: the refusal comes before anything is launched)"""
    from train_gpt_b200._lib import TG_ERR_ALIGN, TG_ERR_SHAPE, TG_ERR_TOO_LARGE, TG_OK, DistillArgs
    p = [4096 * i for i in range(1, 18)]

    def top(logits=p[0], cap=15.0, t=1.0, ids=p[1], rows=4, vocab=100, ld=100, k=5):
        return lib.tg_top_logits(logits, cap, t, ids, p[2], p[3], rows, vocab, ld, k, None)

    assert top(ld=99) == top(k=0) == top(k=101) == top(ids=None) == top(cap=65.0) == top(t=0.1) == top(rows=-1) == TG_ERR_SHAPE
    assert top(vocab=1000, ld=1000, k=257) == top(vocab=2 ** 20 + 1, ld=2 ** 21) == top(rows=2 ** 31) == TG_ERR_TOO_LARGE
    assert top(logits=4097) == TG_ERR_ALIGN and top(rows=0) == TG_OK

    def distill(**kw):
        a = dict(logits=p[0], ids=p[1], logp=p[2], targets=p[3], cap=15.0, temperature=1.0, weight=0.5, dlogits=p[4], row_loss=p[5], rows=4, vocab=100, ld=100, k=5)
        a.update(kw)
        return lib.tg_softcap_distill(ctypes.byref(DistillArgs(**a)), None)

    assert distill(ld=99) == distill(ids=None) == distill(logp=None) == distill(k=-1) == distill(weight=1.5) == distill(cap=0.0) == TG_ERR_SHAPE
    assert distill(only_if_scaled=1) == distill(dlogits=None, row_loss=None) == distill(temperature=0.0) == TG_ERR_SHAPE
    assert distill(k=257) == distill(vocab=2 ** 20 + 1, ld=2 ** 21) == TG_ERR_TOO_LARGE
    assert distill(dlogits=p[4] + 2) == distill(logits=4097) == TG_ERR_ALIGN and distill(rows=0) == TG_OK
    assert lib.tg_softcap_distill(None, None) == TG_ERR_SHAPE

    def fwd(x=p[0], gate=p[4], kind=1, x_new=p[5], h=p[6], q=None, s=None, rows=4, cols=256):
        return lib.tg_sandwich_norm_fwd(x, p[1], p[2], p[3], gate, kind, 1.0, 1e-5, x_new, h, q, s, rows, cols, None)

    assert fwd(cols=100) == fwd(gate=None) == fwd(kind=3) == fwd(x_new=None) == fwd(h=None) == fwd(q=p[7]) == fwd(q=p[7], s=p[8], cols=264) == TG_ERR_SHAPE
    assert fwd(cols=8200) == TG_ERR_TOO_LARGE and fwd(x=p[0] + 8) == fwd(gate=p[4] + 2) == TG_ERR_ALIGN and fwd(rows=0) == TG_OK

    def bwd(g=p[5], gate=p[4], kind=1, dpost=p[9], cols=256, scratch=p[12]):
        return lib.tg_sandwich_norm_bwd(p[0], p[1], p[2], p[3], gate, kind, 1.0, 1e-5, g, p[6], p[7], p[8], dpost, p[10], p[11], scratch, 4, cols, None)

    assert bwd(cols=100) == bwd(dpost=None) == bwd(gate=None) == bwd(kind=-1) == TG_ERR_SHAPE
    assert bwd(cols=8200) == TG_ERR_TOO_LARGE and bwd(g=p[5] + 2) == bwd(scratch=p[12] + 8) == TG_ERR_ALIGN
    assert lib.tg_sandwich_norm_bwd_scratch_bytes(0, 256) == 0 == lib.tg_sandwich_norm_bwd_scratch_bytes(4, 9000)

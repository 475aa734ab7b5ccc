"""Pointers that the C entries of the distillation operators and of the sandwich norm cannot do without, and outputs that would lie on their
inputs: refused with a status before any device work."""
import ctypes

import pytest

ADDRESS = [1 << 20 | 4096 * i for i in range(1, 18)]     # aligned numbers that stand for addresses; no call here gets as far as a launch


@pytest.fixture(scope="module")
def lib():
    from train_gpt_b200 import _lib, build
    build.build()
    return _lib.load()


def test_top_logits_without_logits(lib):
    from train_gpt_b200._lib import TG_ERR_SHAPE, TG_OK
    p = ADDRESS
    assert lib.tg_top_logits(None, 15.0, 1.0, p[1], p[2], p[3], 4, 100, 100, 5, None) == TG_ERR_SHAPE
    assert lib.tg_top_logits(None, 15.0, 1.0, p[1], p[2], p[3], 0, 100, 100, 5, None) == TG_OK


def _distill(lib, **kw):
    from train_gpt_b200._lib import DistillArgs
    p = ADDRESS
    a = dict(logits=p[0], ids=p[1], logp=p[2], targets=p[3], cap=15.0, temperature=1.0, weight=0.5, dlogits=p[4], row_loss=p[5], rows=4, vocab=100, ld=100, k=5)
    a.update(kw)
    return lib.tg_softcap_distill(ctypes.byref(DistillArgs(**a)), None)


def test_distillation_without_logits(lib):
    from train_gpt_b200._lib import TG_ERR_SHAPE, TG_OK
    assert _distill(lib, logits=None) == _distill(lib, logits=None, dlogits=None) == TG_ERR_SHAPE
    assert _distill(lib, logits=None, rows=0) == TG_OK


@pytest.mark.parametrize("elements,rows,vocab,ld", [
    (0, 4, 100, 100),                       # the logits' own buffer
    (0, 1, 1, 1),
    (96, 1, 100, 100),                      # the end of the only row
    (-96, 1, 100, 100),
    (296, 4, 100, 100),                     # the last row alone
    (-296, 4, 100, 100),
    (96, 4, 100, 200),                      # rows with a pitch: the end of each
    (128, 4, 100, 200),                     # and the beginning of the next one
    (-128, 4, 100, 200),
    (720, 4, 100, 216),                     # three rows further, from 72 on
])
def test_gradient_over_the_logits(lib, elements, rows, vocab, ld):
    from train_gpt_b200._lib import TG_ERR_SHAPE
    assert _distill(lib, dlogits=ADDRESS[0] + 2 * elements, rows=rows, vocab=vocab, ld=ld) == TG_ERR_SHAPE


@pytest.mark.parametrize("missing", ["x", "branch"])
def test_sandwich_forward(lib, missing):
    from train_gpt_b200._lib import TG_ERR_SHAPE, TG_OK
    p = dict(zip(("x", "branch", "post", "pre"), ADDRESS))
    p[missing] = None

    def call(rows):
        return lib.tg_sandwich_norm_fwd(p["x"], p["branch"], p["post"], p["pre"], None, 0, 1.0, 1e-5, ADDRESS[5], ADDRESS[6], None, None, rows, 256, None)
    assert call(4) == TG_ERR_SHAPE and call(0) == TG_OK


@pytest.mark.parametrize("missing", ["x_new", "branch", "dx", "dbranch", "scratch"])
def test_sandwich_backward(lib, missing):
    from train_gpt_b200._lib import TG_ERR_SHAPE
    names = ("x_new", "branch", "post", "pre", "g_new", "g_h", "dx", "dbranch", "dpost", "dpre", "scratch")
    p = dict(zip(names, ADDRESS))
    p[missing] = None
    assert lib.tg_sandwich_norm_bwd(p["x_new"], p["branch"], p["post"], p["pre"], None, 0, 1.0, 1e-5, p["g_new"], p["g_h"], p["dx"], p["dbranch"],
                                    p["dpost"], p["dpre"], None, p["scratch"], 4, 256, None) == TG_ERR_SHAPE

"""What the norm and rotation of queries and keys, the gated projections and the dropout refuse, checked where it is refused: on the host, before
any device work.  And the generator's known answers."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import block_reference as ref

BF = torch.bfloat16
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype)


@pytest.fixture(scope="module")
def lib():
    from train_gpt_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("q,k,kw,message", [
    ((2, 3, 4, 64), (2, 3, 4, 32), {}, "do not match"),
    ((2, 3, 4, 64), (2, 4, 4, 64), {}, "do not match"),
    ((2, 3, 4, 64), (3, 4, 64), {}, "must be"),
    ((64,), (64,), {}, "must be"),
    ((2, 3, 4, 40), (2, 3, 4, 40), {}, "dim=40"),
    ((2, 3, 4, 528), (2, 3, 4, 528), {}, "dim=528"),
    ((2, 3, 4, 0), (2, 3, 4, 0), {}, "dim=0"),
    ((2, 3, 0, 64), (2, 3, 4, 64), {}, "must have heads"),
    ((2, 3, 4, 64), (2, 3, 4, 64), dict(rotary_dim=8), "rotary_dim=8"),
    ((2, 3, 4, 64), (2, 3, 4, 64), dict(rotary_dim=80), "rotary_dim=80"),
    ((2, 3, 4, 64), (2, 3, 4, 64), dict(rotary_dim=-16), "rotary_dim=-16"),
    ((2, 3, 4, 64), (2, 3, 4, 64), dict(theta=0.0), "theta="),
    ((2, 3, 4, 64), (2, 3, 4, 64), dict(theta=float("nan")), "theta="),
])
def test_rope_shapes(q, k, kw, message):
    from train_gpt_b200 import kernels
    with pytest.raises(ValueError, match=message):
        kernels.qk_norm_rope(_z(*q), _z(*k), None, None, 1e-5, **kw)


def test_rope_scales():
    from train_gpt_b200 import kernels
    q = _z(2, 3, 4, 64)
    with pytest.raises(ValueError, match="both or neither"):
        kernels.qk_norm_rope(q, q, _z(64), None, 1e-5)
    with pytest.raises(ValueError, match="scale shape"):
        kernels.qk_norm_rope(q, q, _z(64), _z(32), 1e-5)


def test_no_cpu_path():
    from train_gpt_b200 import kernels
    q = _z(2, 3, 4, 64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.qk_norm_rope(q, q, None, None, 1e-5)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.gated_linear(_z(2, 8), _z(8, 16), _z(8, 16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.dropout(_z(8), 0.5, _z(1, dtype=torch.int64))


@pytest.mark.parametrize("x,g,u,message", [
    ((4, 16), (16, 8), (16, 16), "one shape"), ((4, 16), (16,), (16,), "one shape"), ((4, 16), (8, 8), (8, 8), "contracted-dim mismatch"),
    ((4, 12), (12, 8), (12, 8), "multiples of 8"), ((4, 16), (16, 12), (16, 12), "multiples of 8"), ((4, 16), (16, 0), (16, 0), "multiples of 8"),
    ((), (16, 8), (16, 8), "at least one dimension"),
])
def test_gated_shapes(x, g, u, message):
    from train_gpt_b200 import kernels
    with pytest.raises(ValueError, match=message):
        kernels.gated_linear(_z(*x), _z(*g), _z(*u))


def test_gated_activation():
    from train_gpt_b200 import kernels
    with pytest.raises(ValueError, match="unknown activation 'tanh'"):
        kernels.gated_linear(_z(4, 16), _z(16, 8), _z(16, 8), "tanh")


@pytest.mark.parametrize("kw,message", [
    (dict(p=-0.1), "p="), (dict(p=1.5), "p="), (dict(p=float("nan")), "p="), (dict(site=-1), "site="), (dict(site=2 ** 32), "site="),
    (dict(residual=_z(9)), "residual shape"), (dict(seed=_z(2, dtype=torch.int64)), "one number"), (dict(seed=_z(0, dtype=torch.int64)), "one number"),
])
def test_dropout_arguments(kw, message):
    from train_gpt_b200 import kernels
    args = dict(p=0.5, seed=_z(1, dtype=torch.int64), site=0, residual=None)
    args.update(kw)
    with pytest.raises(ValueError, match=message):
        kernels.dropout(_z(8), **args)


# ---- the C entries: aligned numbers stand for addresses, nothing is launched ---------------------------------------

A = [4096 * (i + 1) for i in range(20)]


def _qk(**kw):
    from train_gpt_b200._lib import QkArgs
    s = (3 * 4 * 64, 4 * 64, 64)
    a = QkArgs(q=A[0], k=A[1], q_stride=s, k_stride=s, q_out=A[2], k_out=A[3], q_scale=A[4], k_scale=A[5], batch=2, tokens=3, heads=4, kv_heads=4, dim=64, rotary_dim=64,
               eps=1e-5, theta=1e4, g_q=A[6], g_k=A[7], g_q_stride=s, g_k_stride=s, dq_scale=A[8], dk_scale=A[9], scratch=A[10])
    for n, v in kw.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_rope_entries(lib):
    from train_gpt_b200._lib import TG_ERR_ALIGN, TG_ERR_SHAPE, TG_ERR_TOO_LARGE, TG_OK
    both = (lib.tg_qk_norm_rope_fwd, lib.tg_qk_norm_rope_bwd)
    s = (ctypes.c_int64 * 3)
    for kw in (dict(dim=40), dict(dim=0), dict(rotary_dim=8), dict(rotary_dim=80), dict(rotary_dim=-16), dict(heads=0), dict(kv_heads=0), dict(theta=0.0),
               dict(theta=float("nan")), dict(theta=float("inf")), dict(batch=-1), dict(tokens=-1), dict(q_scale=None), dict(k_scale=None), dict(q_out=None), dict(k_out=None)):
        assert [f(_qk(**kw), None) for f in both] == [TG_ERR_SHAPE] * 2, kw
    for kw in (dict(dim=528, rotary_dim=0), dict(batch=2 ** 20, tokens=2 ** 20), dict(heads=65537)):
        assert [f(_qk(**kw), None) for f in both] == [TG_ERR_TOO_LARGE] * 2, kw
    for kw in (dict(q=A[0] + 2), dict(k_out=A[3] + 8), dict(q_scale=A[4] + 2), dict(q_stride=s(768, 260, 64)), dict(k_stride=s(768, 256, 4))):
        assert [f(_qk(**kw), None) for f in both] == [TG_ERR_ALIGN] * 2, kw
    for kw in (dict(q=None), dict(k=None)):
        assert [f(_qk(**kw), None) for f in both] == [TG_ERR_SHAPE] * 2, kw
    for kw in (dict(g_q=None), dict(g_k=None), dict(dq_scale=None), dict(dk_scale=None), dict(scratch=None)):
        assert lib.tg_qk_norm_rope_bwd(_qk(**kw), None) == TG_ERR_SHAPE, kw
    for kw in (dict(g_q=A[0] + 2), dict(scratch=A[0] + 4), dict(g_k_stride=s(768, 256, 4))):
        assert lib.tg_qk_norm_rope_bwd(_qk(**kw), None) == TG_ERR_ALIGN, kw
    assert lib.tg_qk_norm_rope_fwd(_qk(batch=0), None) == TG_OK and lib.tg_qk_norm_rope_fwd(None, None) == TG_ERR_SHAPE
    assert lib.tg_qk_norm_rope_bwd_scratch_bytes(_qk(batch=0)) == 0 == lib.tg_qk_norm_rope_bwd_scratch_bytes(_qk(q_scale=None, k_scale=None))
    assert lib.tg_qk_norm_rope_bwd_scratch_bytes(_qk()) > 0


def _gated(**kw):
    from train_gpt_b200._lib import GatedArgs
    a = GatedArgs(x=A[0], ldx=64, w_gate=A[1], ld_gate=72, w_up=A[2], ld_up=72, act=0, h=A[3], saved_gate=A[4], saved_up=A[5], saved_exponents=A[6], g=A[7], dx=A[8],
                  dw_gate=A[9], dw_up=A[10], scratch=A[11], scratch_bytes=2 * 1536, rows=10, cols=64, inner=72)
    for n, v in kw.items():
        setattr(a, n, v)
    return ctypes.byref(a)


def test_gated_entries(lib):
    from train_gpt_b200._lib import TG_ERR_ALIGN, TG_ERR_SHAPE, TG_ERR_TOO_LARGE, TG_OK
    both = (lib.tg_gated_linear_fwd, lib.tg_gated_linear_bwd)
    for kw in (dict(rows=-1), dict(cols=60), dict(inner=60), dict(cols=0), dict(inner=0), dict(act=3), dict(act=-1), dict(ldx=56), dict(ld_gate=64), dict(ld_up=64),
               dict(saved_gate=None), dict(saved_up=None), dict(saved_exponents=None), dict(x=None), dict(w_gate=None), dict(w_up=None)):
        assert [f(_gated(**kw), None) for f in both] == [TG_ERR_SHAPE] * 2, kw
    for kw in (dict(rows=2 ** 30 + 1), dict(cols=2 ** 26 + 8, ldx=2 ** 26 + 8), dict(inner=2 ** 26 + 8, ld_gate=2 ** 27, ld_up=2 ** 27), dict(rows=2 ** 30, inner=2 ** 26, ld_gate=2 ** 26, ld_up=2 ** 26)):
        assert [f(_gated(**kw), None) for f in both] == [TG_ERR_TOO_LARGE] * 2, kw
    for kw in (dict(x=A[0] + 2), dict(w_up=A[0] + 8), dict(ldx=68), dict(ld_gate=76), dict(saved_gate=A[0] + 2), dict(saved_exponents=A[0] + 1)):
        assert [f(_gated(**kw), None) for f in both] == [TG_ERR_ALIGN] * 2, kw
    assert lib.tg_gated_linear_fwd(_gated(h=None), None) == TG_ERR_SHAPE and lib.tg_gated_linear_fwd(_gated(h=A[0] + 2), None) == TG_ERR_ALIGN
    for kw in (dict(g=None), dict(scratch=None), dict(scratch_bytes=2 * 1536 - 1), dict(dw_gate=None), dict(dw_up=None)):
        assert lib.tg_gated_linear_bwd(_gated(**kw), None) == TG_ERR_SHAPE, kw
    for kw in (dict(g=A[0] + 2), dict(scratch=A[0] + 4), dict(dx=A[0] + 2), dict(dw_up=A[0] + 2)):
        assert lib.tg_gated_linear_bwd(_gated(**kw), None) == TG_ERR_ALIGN, kw
    assert lib.tg_gated_linear_fwd(_gated(rows=0), None) == TG_OK and lib.tg_gated_linear_fwd(None, None) == TG_ERR_SHAPE
    assert lib.tg_gated_linear_exponent_bytes(10, 72) == 2 * 10 * 2 and lib.tg_gated_linear_exponent_bytes(0, 72) == 0
    assert lib.tg_gated_linear_bwd_scratch_bytes(_gated()) == 2 * (2 * 64 * 72 * 2)          # (in two pieces, 64 rows apart)
    assert lib.tg_gated_linear_bwd_scratch_bytes(_gated(rows=0)) == 0
    long = dict(rows=65536, cols=512, ldx=512, inner=64, ld_gate=64, ld_up=64)      # four tiles of the weights' gradients, of 1024 stages
    assert lib.tg_gated_linear_bwd_scratch_bytes(_gated(**long)) > 2 * 65536 * 128
    assert lib.tg_gated_linear_bwd_scratch_bytes(_gated(**long, dw_gate=None, dw_up=None)) == 2 * 65536 * 128


def test_dropout_entry(lib):
    from train_gpt_b200._lib import TG_ERR_ALIGN, TG_ERR_SHAPE, TG_OK

    def call(x=A[0], residual=A[1], p=0.5, seed=A[2], y=A[3], n=100):
        return lib.tg_dropout(x, residual, p, seed, 0, y, n, None)
    for kw in (dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(n=-1), dict(x=None), dict(y=None), dict(seed=None)):
        assert call(**kw) == TG_ERR_SHAPE, kw
    for kw in (dict(x=A[0] + 2), dict(y=A[0] + 8), dict(residual=A[0] + 4), dict(seed=A[0] + 4)):
        assert call(**kw) == TG_ERR_ALIGN, kw
    assert call(n=0) == TG_OK


def test_structs_have_the_headers_layout():
    from train_gpt_b200._lib import GatedArgs, QkArgs
    assert QkArgs.positions.offset == 8 * 12 and QkArgs.batch.offset == 8 * 16 and QkArgs.theta.offset == 8 * 21 and ctypes.sizeof(QkArgs) == 8 * 33
    assert GatedArgs.h.offset == 56 and GatedArgs.rows.offset == 8 * 17 and ctypes.sizeof(GatedArgs) == 8 * 21


# ---- the generator ----------------------------------------------------------------------------------------------------

def test_known_answers_of_the_generator():
    """Philox4x32-10's published ones: all zeros, all ones, digits of pi."""
    for counter, key, want in (((0,) * 4, (0,) * 2, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"), ((0xFFFFFFFF,) * 4, (0xFFFFFFFF,) * 2, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), "d16cfe09 94fdcceb 5001e420 24126ea1")):
        assert " ".join(f"{v:08x}" for v in ref.philox(np.array([counter], dtype=np.uint64), key)[0]) == want


# ---- rules that no run can be relied on to test --------------------------------------------------------------------

def test_the_pairs_kernel_keeps_the_gemms_rules():
    """As test_tensor_memory_source and test_warp_order_source for the other GEMMs: dependents start after the allocation, nothing is read
    before the wait for the kernel before, an arrival for a whole warp follows its __syncwarp."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(ROOT, "train_gpt_b200", "csrc", "gated.cu")).read())
    pairs, few = text[text.index("void gated_body("):text.index("gated_fwd_kernel(")], text[text.index("gated_few_kernel(const"):text.index("struct GatedSlopes")]
    for body, take, meet, touch in ((pairs, "tmem_take_pair(", "cluster_sync();", ("tma_load", "tma_store", "exponents")), (few, "tmem_take(", "__syncthreads();", ("tma_load", "few_join<"))):
        taken = body.index(take)
        met, trigger, wait = (body.index(s, taken) for s in (meet, "grid_trigger();", "grid_wait();"))
        assert taken < met < trigger < wait < min(body.index(s) for s in touch)
        assert body.count("grid_trigger();") == body.count("grid_wait();") == 1
    arrivals = list(re.finditer(r"\bmbar_arrive(?:_cluster)?_if\(", pairs))
    assert arrivals and "mbar_arrive" not in few
    for m in arrivals:
        marks = re.findall(r"__syncwarp\(\);|__all_sync\(|\bmbar_wait\(|\btmem_wait_ld\w*\(", pairs[:m.start()])
        assert marks[-1] == "__syncwarp();"

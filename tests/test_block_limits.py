"""Limits of the block's operators that are refused on the host, before any device work; aligned numbers stand for addresses."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from train_gpt_b200 import _lib, build
    build.build()
    return _lib.load()


@pytest.mark.parametrize("theta", [1e-300, 5e-324, 9e-31, -1.0])
def test_bases_whose_angles_are_no_numbers(lib, theta):
    """From 1e-30 on a far token's is finite whatever is rotated; of the smallest doubles its angle goes past the largest."""
    from train_gpt_b200 import kernels
    from train_gpt_b200._lib import TG_ERR_SHAPE, QkArgs
    q = torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="theta="):
        kernels.qk_norm_rope(q, q, None, None, 1e-5, theta=theta)
    s = (768, 256, 64)
    a = QkArgs(q=4096, k=8192, q_stride=s, k_stride=s, q_out=12288, k_out=16384, batch=2, tokens=3, heads=4, kv_heads=4, dim=64, rotary_dim=64, theta=theta, g_q=20480,
               g_k=24576, g_q_stride=s, g_k_stride=s)
    assert lib.tg_qk_norm_rope_fwd(ctypes.byref(a), None) == lib.tg_qk_norm_rope_bwd(ctypes.byref(a), None) == TG_ERR_SHAPE


def _gated(rows, scratch_bytes, **kw):
    from train_gpt_b200._lib import GatedArgs
    a = [4096 * (i + 1) for i in range(12)]
    g = GatedArgs(x=a[0], ldx=8, w_gate=a[1], ld_gate=8, w_up=a[2], ld_up=8, act=0, h=a[3], saved_gate=a[4], saved_up=a[5], saved_exponents=a[6], g=a[7], dx=a[8], dw_gate=a[9],
                  dw_up=a[10], scratch=a[11], scratch_bytes=scratch_bytes, rows=rows, cols=8, inner=8)
    for n, v in kw.items():
        setattr(g, n, v)
    return ctypes.byref(g)


def test_rows_of_the_weights_gradients_with_the_least_scratch(lib):
    """One item's stages have a limit, 2^27 rows, that the ranges of the whole scratch keep: the refusal needs no device."""
    from train_gpt_b200._lib import TG_ERR_ARCH, TG_ERR_CUDA, TG_ERR_TOO_LARGE
    for rows in (2 ** 27 + 64, 2 ** 30):
        least = 2 * rows * 16
        assert lib.tg_gated_linear_bwd(_gated(rows, least), None) == TG_ERR_TOO_LARGE
        assert lib.tg_gated_linear_bwd_scratch_bytes(_gated(rows, 0)) > least
    if not torch.cuda.is_available():               # (what is not refused would be launched: without a device it fails behind the checks)
        for rows, scratch, kw in ((2 ** 27, 2 ** 32, {}), (2 ** 30, 2 ** 35, dict(dw_gate=None, dw_up=None)),
                                  (2 ** 30, lib.tg_gated_linear_bwd_scratch_bytes(_gated(2 ** 30, 0)), {})):
            assert lib.tg_gated_linear_bwd(_gated(rows, scratch, **kw), None) in (TG_ERR_ARCH, TG_ERR_CUDA), (rows, kw)


@pytest.mark.parametrize("rows,cols,inner,want", [(65536, 512, 64, 63963136), (2 ** 20, 64, 64, 315621376), (2 ** 20, 1024, 64, 316669952), (2 ** 24, 64, 64, 4341628928),
                                                  (2 ** 27, 64, 64, 34406400000), (128, 128, 512, 1048576), (32768, 1024, 4096, 536870912)])
def test_the_plans_of_long_contractions(lib, rows, cols, inner, want):
    """The search for the best order of two problems looks no further than where the second has been taken up whole: these are the plans that it made when it did."""
    a = _gated(rows, 0, cols=cols, ldx=cols, inner=inner, ld_gate=inner, ld_up=inner)
    assert lib.tg_gated_linear_bwd_scratch_bytes(a) == want

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

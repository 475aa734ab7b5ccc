"""As many rows as the distillation loss takes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_the_largest_number_of_rows():
    """2^31 - 1 rows of two equal logits: each loss is log 2 (a sum, a logarithm and a difference of values below 2^0, 2^-22 in all)."""
    from train_gpt_b200 import ops
    rows = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GB")
    x = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda")
    targets = torch.zeros(rows, dtype=torch.int32, device="cuda")
    ids, logp = torch.zeros(rows, 0, dtype=torch.int32, device="cuda"), torch.zeros(rows, 0, device="cuda")
    loss, _ = ops.softcap_distill(x, ids, logp, None, 15.0, targets, 1.0, 0.0, want_grad=False)
    low, high = loss.aminmax()
    assert abs(float(low) - math.log(2)) <= 2.0 ** -22 and abs(float(high) - math.log(2)) <= 2.0 ** -22

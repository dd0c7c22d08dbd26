"""CPU: settings of fused_sample that do not fit the call's types are refused."""

import pytest
import torch

from metal_liger_b200.ops.fused_sampling import fused_sample


@pytest.mark.parametrize("k", [2 ** 63, 2 ** 64 + 1])
def test_top_k_past_int64_is_refused(k):
    """It would wrap: 2^64 + 1 to a top_k of 1."""
    with pytest.raises(ValueError, match="top_k"):
        fused_sample(torch.zeros(1, 8), torch.zeros(1), top_k=k)


def test_the_largest_top_k_is_taken():
    with pytest.raises(NotImplementedError):                     # there is no CPU kernel
        fused_sample(torch.zeros(1, 8), torch.zeros(1), top_k=2 ** 63 - 1)

"""-m gpu: sizes beyond what the C ABI's 32-bit fields hold raise the library's error, like every other refusal."""
import pytest
import torch

from muzero_amd import capi, ops

pytestmark = pytest.mark.gpu


def test_sizes_beyond_32_bits():
    long = torch.empty(1, 2**31, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(capi.MuZeroError, match="sizes"):
        ops.sample_actions(long, torch.zeros(1, dtype=torch.float64, device="cuda"))
    index = torch.zeros(1, dtype=torch.int32, device="cuda")
    b = torch.zeros(1, 1, 1, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(capi.MuZeroError, match="sizes"):
        ops.adapter_linear(long, long, long[None], b, index)

"""-m gpu: one row among the wide rows of another operand: beside its columns allowed, over them refused."""
import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests.test_gpu_adapter import check as check_adapter
from tests.test_gpu_adapter import make
from tests.test_gpu_sample import check as check_sample
from tests.test_gpu_sample import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("row", [0, 7, 23])
def test_one_result_row_beside_the_weights(row):
    s = make(np.random.default_rng(row), 1, 64, 24, 4, 3, "bf16")
    wide = torch.zeros(24, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 16:80] = s["weight"]
    s["weight"] = wide[:, 16:80]
    for at in (80, 104):
        check_adapter(s, "bf16", out=wide[row : row + 1, at : at + 24])
    for at in (0, 8, 30, 79):
        with pytest.raises(capi.MuZeroError, match="overlaps"):
            ops.adapter_linear(**s, out=wide[row : row + 1, at : at + 24])


def test_results_beside_one_x_for_all_rows():
    s = make(np.random.default_rng(1), 9, 64, 24, 4, 3, "bf16")
    wide = torch.zeros(9, 128, dtype=torch.bfloat16, device="cuda")
    wide[4, 16:80] = s["x"][0]
    s["x"] = wide[4:5, 16:80].expand(9, 64)
    check_adapter(s, "bf16", out=wide[:, 80:104])
    with pytest.raises(capi.MuZeroError, match="overlaps"):
        ops.adapter_linear(**s, out=wide[:, 60:84])
    check_adapter(s, "bf16", out=wide[:4].reshape(-1)[:216].view(9, 24))     # rows before it


def test_probabilities_of_one_row():
    z, u, _ = inputs(np.random.default_rng(2), 1, 30, torch.float32)
    wide = torch.zeros(1, 64, device="cuda")
    wide[:, :30] = z
    new = lambda p: dict(action=torch.empty(1, dtype=torch.int32, device="cuda"), logprob=torch.empty(1, device="cuda"),  # noqa: E731
                         kept=torch.empty(1, dtype=torch.int32, device="cuda"), probs=p)
    check_sample(wide[:, :30], u, out=new(wide[:, 30:60]))
    with pytest.raises(capi.MuZeroError, match="overlaps"):
        ops.sample_actions(wide[:, :30], u, out=new(wide[:, 29:59]))

"""-m gpu: an error that an earlier HIP call of the thread has left behind is not the operators' own."""
import ctypes as C

import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests.test_gpu_adapter import check as check_adapter
from tests.test_gpu_adapter import make
from tests.test_gpu_policy_moves import context, positions
from tests.test_gpu_sample import check as check_sample
from tests.test_gpu_sample import inputs

pytestmark = pytest.mark.gpu


def leave_an_error():
    """A refused call, whose error stays until someone asks for it."""
    hip = C.CDLL("libamdhip64.so", mode=C.RTLD_GLOBAL)
    assert hip.hipSetDevice(4096) != 0
    return hip


@pytest.mark.parametrize("M", [1, 40, 1200])
def test_projection(M):
    s = make(np.random.default_rng(M), M, 64, 520, 4, 3, "bf16")
    want = check_adapter(s, "bf16")
    out = torch.zeros_like(want)
    workspace = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    hip = leave_an_error()
    ops.adapter_linear(**s, out=out, workspace=workspace)
    assert hip.hipGetLastError() != 0      # nobody's business here, still there for whoever asks
    assert torch.equal(out, want)


@pytest.mark.parametrize("A", [9, 300, 50000])
def test_sampling(A):
    z, u, _ = inputs(np.random.default_rng(A), 3, A, torch.float32)
    want, _ = check_sample(z, u, top_k=5)
    out = {k: torch.zeros_like(v) for k, v in want.items()}
    workspace = torch.empty(1 << 22, dtype=torch.uint8, device="cuda")
    hip = leave_an_error()
    ops.sample_actions(z, u, top_k=5, out=out, workspace=workspace)
    assert hip.hipGetLastError() != 0
    for k in want:
        assert torch.equal(out[k], want[k])


@pytest.mark.parametrize("precision", [capi.PRECISION_FP32, capi.PRECISION_F16])
def test_raw_policy_moves(precision):
    rng = np.random.default_rng(0)
    spec, _, ctx = context("tictactoe", precision, 4)
    obs, legal, u = positions(rng, spec, 4)
    want = ctx.play_policy(4, obs, legal, u)
    hip = leave_an_error()
    got = ctx.play_policy(4, obs, legal, u)
    hip.hipGetLastError()
    for k in want:
        np.testing.assert_array_equal(got[k], want[k])
    ctx.close()

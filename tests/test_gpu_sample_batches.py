"""-m gpu: ops.sample_actions where the number of rows chooses the kernel, and the kernel pair that shares a row out over workgroups
inside graphs.  The order of the 64-bit sums goes by the kernel, so two batch sizes agree in action and count unless u or top_p lies
within 1e-13 of a border, which these random numbers do not, and in logprob and probs to the rounding of nearly equal numbers to
fp32: one step, 2^-23 of the value (logprob: and 1e-11 for the difference of its two terms)."""
import numpy as np
import pytest
import torch

from muzero_amd import ops
from tests.test_gpu_sample import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,A,f", [(512, 9000, dict(top_p=0.9)), (512, 9000, dict()), (300, 16000, dict(top_k=400, top_p=0.95)),
                                   (150, 60000, dict(top_k=50, top_p=0.9)), (150, 60000, dict(top_p=0.8)), (40, 60000, dict(min_p=0.02))])
def test_a_batch_and_its_rows_alone(B, A, f):
    z, u, legal = inputs(np.random.default_rng(A + B), B, A, torch.bfloat16, mask="legal")
    a = ops.sample_actions(z, u, legal=legal, probs=True, **f)
    for i in range(0, B, B // 9):
        c = ops.sample_actions(z[i : i + 1], u[i : i + 1], legal=legal[i : i + 1], probs=True, **f)
        for k in ("action", "kept"):
            assert torch.equal(a[k][i : i + 1], c[k]), (k, i)
        torch.testing.assert_close(a["logprob"][i : i + 1], c["logprob"], rtol=2.0**-23, atol=1e-11)
        torch.testing.assert_close(a["probs"][i : i + 1], c["probs"], rtol=2.0**-23, atol=2.0**-149)


@pytest.mark.parametrize("B,A", [(1, 131072), (4, 50257), (40, 50000), (100, 98304)])
def test_graph_replays_of_shared_rows(B, A):
    rng = np.random.default_rng(B)
    f, second = dict(top_k=50, top_p=0.95), dict(min_p=0.05, temperature=0.6)
    z, u, legal = inputs(rng, B, A, torch.float16, mask="legal")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_actions(z, u, legal=legal, **f)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ops.sample_actions(z, u, legal=legal, **f)
    with torch.cuda.graph(g2):
        o2 = ops.sample_actions(z, u, legal=legal, **second)
    for step in range(5):
        for old, new in zip((z, u, legal), inputs(rng, B, A, torch.float16, mask="legal")):
            old.copy_(new)
        for v in (*o1.values(), *o2.values()):
            v.zero_()
        for g in (g1, g2) if step % 2 else (g2, g1, g1):
            g.replay()
        e1, e2 = ops.sample_actions(z, u, legal=legal, **f), ops.sample_actions(z, u, legal=legal, **second)
        torch.cuda.synchronize()
        for k in e1:
            assert torch.equal(o1[k], e1[k]) and torch.equal(o2[k], e2[k]), (step, k)
    if B * A < 10**6:
        check(z, u, legal=legal, **f)

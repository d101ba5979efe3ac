"""-m gpu: ops.sample_actions where the border of a filter lies at zero: zeros of both signs beside subnormal values.  Entries are
counted by an order-preserving key, in which a range may end just below zero, at the key of -0; its zeros belong above that range.
With the maximum at the largest float the first ranges end there, and a temperature of 1e300 makes all weights 1, so sums are exact."""
import numpy as np
import pytest
import torch

from tests.test_gpu_sample import check

pytestmark = pytest.mark.gpu
LARGEST, LEAST = 3.4028234663852886e38, 1.401298464324817e-45


def rows(rng, A):
    """One largest entry, then zeros and subnormals in the shares given, shuffled: the same value, a value each, both signs."""
    z = np.zeros((6, A))
    half = (A - 1) // 2
    z[0, :half] = -1e-40                                      # one value below zero
    z[1, :half] = -LEAST * (1 + np.arange(half))              # a value each
    z[2, :half] = -LEAST * rng.integers(1, 2**21, half)       # all over the range next to zero
    z[3, : 2 * half] = LEAST * rng.integers(-(2**20), 2**20, 2 * half)
    z[4, :half] = -LEAST
    z[4, half : 2 * half] = LEAST
    z[5, :] = -LEAST * rng.integers(1, 300, A)                # and no zero at all
    z[:, -1] = LARGEST
    z = rng.permuted(z, axis=1).astype(np.float32)
    z[:, ::3] = np.where(z[:, ::3] == 0, np.float32(-0.0), z[:, ::3])
    return torch.from_numpy(z).cuda()


@pytest.mark.parametrize("A", [400, 700, 2500, 9001, 50001])
def test_borders_next_to_zero(A):
    rng = np.random.default_rng(A)
    z = rows(rng, A)
    u = torch.from_numpy(rng.uniform(size=len(z))).cuda()
    for f in (dict(top_k=A // 2), dict(top_k=3 * A // 4), dict(top_k=A - 2), dict(top_p=0.5), dict(top_p=0.75), dict(top_p=0.99),
              dict(top_k=3 * A // 4, top_p=0.9), dict(top_k=129)):
        check(z, u, temperature=1e300, **f)
        check(z, u, temperature=1.0, **f)


def test_300_of_400():
    """One largest entry, 199 zeros, 200 of -1e-40: the first 300 end among the latter."""
    z = np.zeros(400, np.float32)
    z[0] = LARGEST
    z[1::2] = -1e-40
    u = torch.from_numpy(np.linspace(0, 1, 16)).cuda()
    got, _ = check(torch.from_numpy(z).cuda().expand(16, 400), u, temperature=1e300, top_k=300)
    assert (got["kept"] == 300).all()

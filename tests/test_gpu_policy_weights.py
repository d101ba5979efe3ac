"""-m gpu: mz_play_policy with adapters plays the network as last loaded or committed, whatever has been written since through
mz_weights_device_ptr."""
import numpy as np
import pytest

from muzero_amd import capi, netspec
from tests.test_gpu_comm_weights import _memcpy_h2d
from tests.test_gpu_policy_moves import adapters, context, positions

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("precision", [capi.PRECISION_FP32, capi.PRECISION_F16])
@pytest.mark.parametrize("name", ["tictactoe", "go9"])
def test_weights_written_but_not_committed(name, precision):
    rng = np.random.default_rng(0)
    B = 9
    spec, w, ctx = context(name, precision, B)
    obs, legal, u = positions(rng, spec, B)
    a, b, scale = adapters(rng, spec, 3, 4)
    ctx.load_policy_adapters(a, b, scale)
    index = rng.integers(-1, 3, B).astype(np.int32)
    play = lambda: [ctx.play_policy(B, obs, legal, u, adapter=i)["logits"] for i in (index, None)]  # noqa: E731
    before = play()
    new = netspec.pack_blob(spec, netspec.random_weights(spec, seed=4, ln_jitter=0.1))
    ptr, nbytes = ctx.weights_device_ptr()
    assert nbytes == new.nbytes
    _memcpy_h2d(ptr, new)
    for x, y in zip(play(), before):
        np.testing.assert_array_equal(x, y)
    ctx.commit_weights()
    committed = play()
    assert (committed[0] != before[0]).any(1).all()
    ctx.load_weights(new)
    for x, y in zip(play(), committed):
        np.testing.assert_array_equal(x, y)
    ctx.close()

"""-m gpu: ops.adapter_linear where rows x outputs make many tiles (sides of 64, 128 and 256), against 64-bit products on the host
with the tolerances of test_gpu_adapter.py.  Few adapters go through the matrix instructions, many by rows."""
import numpy as np
import pytest
import torch

from muzero_amd import ops
from tests.test_gpu_adapter import TYPES, check, make

pytestmark = pytest.mark.gpu
SMALL, MIDDLE, LARGE = (1100, 520), (2100, 2100), (4200, 4200)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K", [1, 2, 3, 7, 8, 15, 16, 31, 32, 33, 48, 64, 65, 96, 128, 160, 200, 257, 1000])
def test_inner_lengths(K, dtype):
    """Every number of stages that the split of K can leave one side without, whole and with a rest, aligned and not."""
    rng = np.random.default_rng(K)
    check(make(rng, *SMALL[:1], K, SMALL[1], 8, 3, dtype), dtype)
    check(make(rng, *SMALL[:1], K, SMALL[1], 5, 12, dtype, bias=False, scale=False, order="runs"), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K", [4, 40, 96, 130, 256])
def test_inner_lengths_of_larger_tiles(K, dtype):
    rng = np.random.default_rng(K + 1)
    check(make(rng, *MIDDLE[:1], K, MIDDLE[1], 8, 3, dtype), dtype)
    check(make(rng, *MIDDLE[:1], K, MIDDLE[1], 12, 20, dtype, order="distinct"), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K,n", [(24, 3), (128, 40), (193, 2)])
def test_largest_tiles(K, n, dtype):
    rng = np.random.default_rng(K + 2)
    check(make(rng, LARGE[0], K, LARGE[1], 9, n, dtype), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("r", [1, 3, 4, 8, 15, 16, 17, 32, 33, 64, 100, 128])
def test_ranks(r, dtype):
    rng = np.random.default_rng(r)
    for n in (2, 30):
        check(make(rng, SMALL[0], 136, SMALL[1], r, n, dtype), dtype)
    check(make(rng, MIDDLE[0], 64, MIDDLE[1], r, 4, dtype), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N", [(1037, 641), (2049, 2177), (65, 8257), (8257, 65), (520, 1100)])
def test_strides_offsets_and_untouched_neighbours(M, N, dtype):
    rng = np.random.default_rng(M + 1)
    for K, off in ((96, 1), (128, 8)):
        s = make(rng, M, K, N, 8, 3, dtype)
        t = TYPES[dtype]
        bx = torch.full((M, K + 24), float("nan"), dtype=t, device="cuda")
        bw = torch.full((N, K + 40), float("nan"), dtype=t, device="cuda")
        bx[:, off : off + K] = s["x"]
        bw[:, off : off + K] = s["weight"]
        s["x"], s["weight"] = bx[:, off : off + K], bw[:, off : off + K]
        wide = torch.full((M + 2, N + 16), 7.0, dtype=t, device="cuda")
        check(s, dtype, out=wide[1 : M + 1, off : off + N])
        wide[1 : M + 1, off : off + N] = 7.0
        assert (wide == 7.0).all()
        s["x"] = s["x"][:1].expand(M, K)        # every row the same x: stride 0
        check(s, dtype, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [SMALL, MIDDLE])
@pytest.mark.parametrize("n", [3, 24])
def test_rows_do_not_influence_one_another(n, shape, dtype):
    """inf / NaN of one row's x, of one adapter or of t stay with the rows that use them; foreign indexes give NaN rows."""
    rng = np.random.default_rng(n)
    M, N = shape
    s = make(rng, M, 96, N, 10, n, dtype)
    s["index"] = torch.from_numpy((np.arange(M) % (n + 1) - 1).astype(np.int32)).cuda()
    s["a"][1, 3, 5] = float("nan")
    s["b"][2, 7, 1] = float("inf")
    s["x"][M - 1, 3] = float("inf")
    s["index"][0] = n
    s["index"][1] = -2
    s["index"][2] = 2**31 - 1
    y = check(s, dtype)
    assert torch.isnan(y[0:3]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_and_small_intermediate_values(dtype):
    """x A^T far outside the range of 16-bit floats, B making up for it."""
    rng = np.random.default_rng(3)
    for up, down in ((6e3, 1e-4), (1e-3, 100.0)):
        for n in (3, 24):
            s = make(rng, SMALL[0], 512, SMALL[1], 8, n, dtype)
            s["x"] *= 4
            s["a"] *= up
            s["b"] *= down
            check(s, dtype)


@pytest.mark.parametrize("n", [3, 24])
@pytest.mark.parametrize("shape", [SMALL, MIDDLE])
def test_twice_and_in_another_batch(shape, n):
    """Bit for bit: the same call again, and a row's result whatever adapters the rows beside it use."""
    rng = np.random.default_rng(n + 3)
    s = make(rng, shape[0], 200, shape[1], 16, n, "bf16")
    a, b = ops.adapter_linear(**s), ops.adapter_linear(**s)
    assert torch.equal(a, b)
    keep = s["index"] == 2
    s["index"] = torch.where(keep, s["index"], torch.flip(s["index"], [0]))
    assert torch.equal(ops.adapter_linear(**s)[keep], a[keep])


def test_two_streams_and_graph_replays():
    """Two calls in flight on streams of their own, and two captured ones replayed in turn with eager calls between."""
    rng = np.random.default_rng(6)
    s, o = (make(rng, *SMALL[:1], 256, SMALL[1], 16, n, "bf16") for n in (5, 24))
    want_s, want_o = ops.adapter_linear(**s), ops.adapter_linear(**o)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        with torch.cuda.stream(one):
            ys = ops.adapter_linear(**s)
        with torch.cuda.stream(two):
            yo = ops.adapter_linear(**o)
        torch.cuda.synchronize()
        assert torch.equal(ys, want_s) and torch.equal(yo, want_o)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        y1 = ops.adapter_linear(**s)
    with torch.cuda.graph(g2):
        y2 = ops.adapter_linear(**o)
    for step in range(4):
        n = make(rng, *SMALL[:1], 256, SMALL[1], 16, 5, "bf16")
        for k in s:
            s[k].copy_(n[k])
        g1.replay()
        g2.replay()
        e1, e2 = ops.adapter_linear(**s), ops.adapter_linear(**o)
        torch.cuda.synchronize()
        assert torch.equal(y1, e1) and torch.equal(y2, e2), step

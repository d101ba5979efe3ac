"""-m gpu: ops.adapter_linear (mz_adapter_linear) against 64-bit products on the host.  Tolerance of one y: an fp32 sum of n terms
is off by at most n steps of 2^-24 of the sum of their absolute values (twice that: the matrix instructions add inside a step in
an order and with roundings of their own; K + rank + 2 terms, the rank's sums being sums of K terms themselves); the rank's
intermediate values enter the second product as two numbers of the inputs' type, 2^-16 (bf16) of their value at worst; and the
result is rounded to its type by half a step."""
import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests import op_refs

pytestmark = pytest.mark.gpu
TYPES = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)
TWO_PARTS = dict(fp32=0.0, bf16=2.0**-16, fp16=2.0**-16)


def make(rng, M, K, N, r, n, dtype, bias=True, scale=True, order="mixed"):
    t = TYPES[dtype]
    dev = lambda v: torch.from_numpy(v.astype(np.float32)).cuda().to(t)  # noqa: E731
    index = rng.integers(-1, n, M).astype(np.int32)
    if order == "distinct":
        index = (np.arange(M) % n).astype(np.int32)
    if order == "runs":
        index = np.sort(index)
    if order == "one":
        index[:] = n - 1
    return dict(x=dev(rng.standard_normal((M, K))), weight=dev(rng.standard_normal((N, K)) / np.sqrt(K)),
                a=dev(rng.standard_normal((n, r, K)) / np.sqrt(K)), b=dev(rng.standard_normal((n, N, r)) / np.sqrt(r)),
                index=torch.from_numpy(index).cuda(), bias=dev(rng.standard_normal(N)) if bias else None,
                scale=torch.from_numpy(rng.uniform(0.2, 2.0, n).astype(np.float32)).cuda() if scale else None)


def check(s, dtype, out=None, out_dtype=None):
    y = ops.adapter_linear(**s, out=out, out_dtype=out_dtype)
    want, size = op_refs.adapter(**s)
    got = y.double().cpu().numpy()
    K, r = s["x"].shape[1], s["a"].shape[1]
    tol = (2 * (K + r + 2) * 2.0**-24 + TWO_PARTS[dtype]) * size
    tol = tol + (torch.finfo(y.dtype).eps / 2) * (np.abs(want) + tol) + torch.finfo(y.dtype).smallest_normal
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isfinite(got), fine)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all()
    off = np.abs(got[fine] - want[fine])
    assert (off <= tol[fine]).all(), ((off > tol[fine]).sum(), (off / tol[fine]).max())
    return y


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 9, 16, 17, 33, 48, 64, 65, 130, 257, 300, 1000])
def test_row_counts(M, dtype):
    rng = np.random.default_rng(M)
    for (K, N, r, n), order in zip(((162, 82, 8, 4), (512, 260, 16, 7), (130, 1000, 5, 3), (1024, 512, 32, 16)),
                                   ("mixed", "distinct", "runs", "one")):
        check(make(rng, M, K, N, r, n, dtype, bias=M % 2 == 0, scale=M % 3 != 0, order=order), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("K", [1, 2, 3, 7, 8, 31, 63, 64, 65, 100, 127, 128, 129, 256, 1000, 2050, 4096])
def test_inner_lengths(K, dtype):
    rng = np.random.default_rng(K)
    for M, N, r, n in ((1, 33, 1, 1), (6, 70, 4, 3), (40, 64, 16, 5), (200, 136, 9, 2)):
        check(make(rng, M, K, N, r, n, dtype), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 15, 16, 17, 63, 64, 65, 82, 255, 256, 257, 1999])
def test_outer_lengths(N, dtype):
    rng = np.random.default_rng(N)
    for M, K, r, n in ((1, 256, 2, 2), (7, 72, 3, 3), (50, 128, 16, 5), (260, 96, 8, 2)):
        check(make(rng, M, K, N, r, n, dtype), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("r", [1, 2, 3, 4, 7, 8, 12, 15, 16, 17, 31, 32, 33, 48, 64, 65, 100, 127, 128])
def test_ranks(r, dtype):
    rng = np.random.default_rng(r)
    for M, K, N, n in ((1, 320, 100, 2), (12, 136, 72, 12), (150, 256, 200, 6)):
        check(make(rng, M, K, N, r, n, dtype, order="distinct" if M == 12 else "mixed"), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,N,r,n", [(1, 4096, 4096, 16, 8), (16, 2048, 8192, 64, 16), (512, 4096, 512, 16, 24),
                                       (2000, 1024, 1024, 16, 64), (4096, 162, 82, 8, 32)])
def test_larger(M, K, N, r, n, dtype):
    rng = np.random.default_rng(M + K)
    for order in ("mixed", "runs"):
        check(make(rng, M, K, N, r, n, dtype, order=order), dtype)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [1, 9, 40, 150])
def test_strides_offsets_and_untouched_neighbours(M, dtype):
    rng = np.random.default_rng(M + 1)
    for K, N, off in ((128, 64, 1), (96, 80, 8), (256, 82, 3), (100, 65, 2)):
        s = make(rng, M, K, N, 8, 3, dtype)
        t = TYPES[dtype]
        bx = torch.full((M, K + 24), float("nan"), dtype=t, device="cuda")
        bw = torch.full((N, K + 40), float("nan"), dtype=t, device="cuda")
        bx[:, off : off + K] = s["x"]
        bw[:, off : off + K] = s["weight"]
        s["x"], s["weight"] = bx[:, off : off + K], bw[:, off : off + K]
        for od in {t, torch.float32}:
            wide = torch.full((M + 2, N + 16), 7.0, dtype=od, device="cuda")
            check(s, dtype, out=wide[1 : M + 1, off : off + N])
            wide[1 : M + 1, off : off + N] = 7.0
            assert (wide == 7.0).all()
        if M > 1:
            s["x"] = s["x"][:1].expand(M, K)        # every row the same x: stride 0
            check(s, dtype, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M", [4, 40, 300])
def test_rows_do_not_influence_one_another(M, dtype):
    """inf / NaN of one row's x or of one adapter stay with the rows that use them; foreign indexes give NaN rows."""
    rng = np.random.default_rng(M + 2)
    s = make(rng, M, 192, 130, 10, 6, dtype)
    s["index"] = torch.from_numpy((np.arange(M) % 7 - 1).astype(np.int32)).cuda()
    s["a"][1, 3, 5] = float("nan")
    s["b"][2, 7, 1] = float("inf")
    s["x"][M - 1, 3] = float("inf")
    s["index"][0] = 6
    s["index"][1] = -2
    s["index"][2] = 2**31 - 1
    y = check(s, dtype)
    assert torch.isnan(y[0:3]).all()


@pytest.mark.parametrize("dtype", list(TYPES))
def test_large_and_small_intermediate_values(dtype):
    """x A^T far outside the range of 16-bit floats, B making up for it."""
    rng = np.random.default_rng(3)
    for M in (2, 100):
        for up, down in ((6e3, 1e-4), (1e-3, 100.0)):
            s = make(rng, M, 512, 96, 8, 3, dtype)
            s["x"] *= 4
            s["a"] *= up
            s["b"] *= down
            check(s, dtype)


@pytest.mark.parametrize("M,order", [(3, "mixed"), (40, "distinct"), (700, "mixed"), (3000, "mixed")])
def test_twice_and_in_another_batch(M, order):
    """Bit for bit: the same call again, and a row's result whatever adapters the rows beside it use."""
    rng = np.random.default_rng(M + 3)
    s = make(rng, M, 512, 256, 16, 8, "bf16", order=order)
    a, b = ops.adapter_linear(**s), ops.adapter_linear(**s)
    assert torch.equal(a, b)
    keep = s["index"] == 2
    s["index"] = torch.where(keep, s["index"], torch.flip(s["index"], [0]))
    assert torch.equal(ops.adapter_linear(**s)[keep], a[keep])


def test_streams_and_graph_replays():
    rng = np.random.default_rng(5)
    for M in (1, 48, 600):
        s = make(rng, M, 256, 192, 16, 5, "bf16")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.adapter_linear(**s)
        torch.cuda.current_stream().wait_stream(side)
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1):
            y1 = ops.adapter_linear(**s)
        with torch.cuda.graph(g2):
            y2 = ops.adapter_linear(**{**s, "scale": None})
        for step in range(4):
            n = make(rng, M, 256, 192, 16, 5, "bf16")
            for k in s:
                s[k].copy_(n[k])
            g1.replay()
            g2.replay()
            e1, e2 = ops.adapter_linear(**s), ops.adapter_linear(**{**s, "scale": None})
            torch.cuda.synchronize()
            assert torch.equal(y1, e1) and torch.equal(y2, e2), step


def test_no_rows_and_refusals_on_the_device():
    s = make(np.random.default_rng(0), 4, 64, 32, 4, 2, "fp32")
    assert ops.adapter_linear(**{**s, "x": s["x"][:0], "index": s["index"][:0]}).shape == (0, 32)
    for change, text in (({"weight": s["weight"].half()}, "weight"), ({"a": s["a"][:, :, :32]}, "a:"), ({"b": s["b"].cpu()}, "b:"),
                         ({"index": s["index"].long()}, "index"), ({"bias": s["bias"][:3]}, "bias"), ({"x": s["x"].t()}, "")):
        with pytest.raises(capi.MuZeroError, match=text or None):
            ops.adapter_linear(**{**s, **change})
    with pytest.raises(capi.MuZeroError, match="gradient"):
        ops.adapter_linear(**{**s, "a": s["a"].clone().requires_grad_()})
    with torch.no_grad():
        ops.adapter_linear(**{**s, "a": s["a"].clone().requires_grad_()})
    with pytest.raises(capi.MuZeroError, match="workspace"):
        ops.adapter_linear(**s, workspace=torch.empty(1, dtype=torch.uint8, device="cuda"))

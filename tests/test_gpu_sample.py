"""-m gpu: ops.sample_actions (mz_sample_actions) against a row-by-row 64-bit restatement.  Actions and counts must be equal.
logprob and probs are 64-bit values rounded once to float32: half a step, 2^-24 of the value, plus the error of the 64-bit sums
(below 1e-12 at these sizes); a logprob is a difference of two numbers below 1e5 in size, whose own rounding is below 1e-11."""
import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests import op_refs

pytestmark = pytest.mark.gpu
TYPES = dict(fp32=torch.float32, bf16=torch.bfloat16, fp16=torch.float16)


def check(logits, u, out=None, **kw):
    got = ops.sample_actions(logits, u, probs=True, out=out, **kw)
    want = op_refs.sample(logits, u, **kw)
    a = {k: v.cpu().numpy() for k, v in got.items()}
    np.testing.assert_array_equal(a["kept"], want["kept"])
    np.testing.assert_array_equal(a["action"], want["action"])
    np.testing.assert_allclose(a["logprob"], want["logprob"], rtol=2.0**-24 + 1e-12, atol=1e-11)
    np.testing.assert_allclose(a["probs"], want["probs"], rtol=2.0**-24 + 1e-11, atol=2.0**-149)
    return got, want


def inputs(rng, B, A, dtype, spread=2.0, mask=None):
    z = torch.from_numpy((spread * rng.standard_normal((B, A))).astype(np.float32)).to(dtype).cuda()
    u = torch.from_numpy(rng.uniform(size=B)).cuda()
    legal = None
    if mask:
        l = rng.uniform(size=(B, A)) < 0.6
        if mask == "empty":
            l[:: 3] = False
        legal = torch.from_numpy(l.astype(np.uint8)).cuda()
        junk = torch.from_numpy(rng.choice([np.nan, np.inf, -np.inf, 3.0e38], size=(B, A)).astype(np.float32)).cuda().to(dtype)
        z = torch.where(legal != 0, z, junk)
    return z, u, legal


FILTERS = dict(none={}, k1=dict(top_k=1), k7=dict(top_k=7), kmany=dict(top_k=200), p=dict(top_p=0.9), pall=dict(top_p=0.99999),
               ptiny=dict(top_p=1e-9), m=dict(min_p=0.05), m1=dict(min_p=1.0), kp=dict(top_k=40, top_p=0.8),
               kbigp=dict(top_k=500, top_p=0.97), kpm=dict(top_k=60, top_p=0.95, min_p=0.02), km=dict(top_k=300, min_p=0.001),
               pm=dict(top_p=0.9, min_p=0.01))


@pytest.mark.parametrize("A", [1, 2, 9, 63, 64, 65, 82, 128, 129, 196, 256, 257, 300, 1000, 4097, 8192, 8193, 20011])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_lengths_and_filters(A, dtype):
    rng = np.random.default_rng(A)
    B = 13 if A <= 1000 else 5
    for i, (name, f) in enumerate(FILTERS.items()):
        z, u, legal = inputs(rng, B, A, TYPES[dtype], mask=[None, "legal", "empty"][i % 3])
        check(z, u, legal=legal, temperature=[1.0, 0.7, 1.9][i % 3], **f)


@pytest.mark.parametrize("A,dtype", [(50257, "fp32"), (131072, "bf16"), (131071, "fp16"), (262144, "fp32")])
def test_long_rows(A, dtype):
    rng = np.random.default_rng(A)
    for i, f in enumerate(FILTERS.values()):
        z, u, legal = inputs(rng, 2, A, TYPES[dtype], spread=[1.0, 3.0][i % 2], mask=[None, "legal"][i % 2])
        check(z, u, legal=legal, temperature=[0.8, 1.3][i % 2], **f)


@pytest.mark.parametrize("A", [40, 200, 700, 9000, 40000])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_ties(A, dtype):
    """Few distinct values: the border falls inside runs of equals, which rank by index.  T = 1 / ln 2 makes the weights powers
    of two, so all sums are exact and borders may be hit exactly."""
    rng = np.random.default_rng(A + 1)
    T = float(1 / np.log(2))
    for f in FILTERS.values():
        z = torch.from_numpy(rng.integers(-3, 4, (4, A)).astype(np.float32)).to(TYPES[dtype]).cuda()
        z[0] = 1.25                                                   # one value
        z[1] = torch.where(torch.arange(A).cuda() % 2 == 0, 0.0, -0.0)   # +0 and -0 are equals
        u = torch.from_numpy(rng.uniform(size=4)).cuda()
        check(z, u, temperature=T * 3.7, **f)


@pytest.mark.parametrize("A", [50, 300, 9001])
def test_extreme_values_and_temperatures(A):
    rng = np.random.default_rng(A + 2)
    for T in (0.0, 5e-324, 1e-30, 1e-3, 1.0, 100.0, 1e30, 1.7e308):
        for f in (dict(), dict(top_k=5), dict(top_k=200), dict(top_p=0.7), dict(min_p=0.3), dict(top_k=20, top_p=0.5, min_p=0.1)):
            z, u, _ = inputs(rng, 12, A, torch.float32)
            z[0, A // 2] = float("inf")
            z[1, :3] = float("inf")
            z[2] = float("-inf")
            z[3] = float("nan")
            z[4] = -3.4028234663852886e38
            z[5, 1:] = -3.4028234663852886e38                       # masks of the type's lowest value
            z[6] *= 1e37
            z[7] = z[7] * 1e-44
            z[8, ::2] = float("nan")
            z[9] = 3.4028234663852886e38
            z[10] += 1e4
            check(z, u, temperature=T, **f)


@pytest.mark.parametrize("A", [5, 82, 256, 400, 9000])
def test_random_numbers_at_the_ends(A):
    rng = np.random.default_rng(A + 3)
    for f in (dict(), dict(top_k=3), dict(top_p=0.6), dict(top_k=150)):
        z, _, legal = inputs(rng, 6, A, torch.float32, mask="legal")
        u = torch.tensor([0.0, 1.0, 1.0 - 2.0**-53, 5e-324, 0.5, 0.0], dtype=torch.float64).cuda()
        check(z, u, legal=legal, **f)


@pytest.mark.parametrize("A", [82, 300, 9000])
def test_per_row_parameters_and_their_refusal(A):
    rng = np.random.default_rng(A + 4)
    B = 64
    z, u, legal = inputs(rng, B, A, torch.float32, mask="empty")
    t = torch.from_numpy(rng.uniform(0.2, 3.0, B)).cuda()
    k = torch.from_numpy(rng.integers(0, 2 * A, B).astype(np.int32)).cuda()
    p = torch.from_numpy(rng.uniform(0.1, 1.0, B)).cuda()
    m = torch.from_numpy(rng.uniform(0.0, 0.3, B)).cuda()
    t[3], t[4], t[5], t[6] = 0.0, -1.0, float("nan"), float("inf")
    k[7], k[8] = -1, 2**31 - 1
    p[9], p[10], p[11] = 0.0, 1.5, float("nan")
    m[12], m[13] = -0.1, 2.0
    u[14], u[15], u[16] = -1e-9, 1.0000001, float("nan")
    got, _ = check(z, u, legal=legal, temperature=t, top_k=k, top_p=p, min_p=m)
    assert (got["action"][[4, 5, 6, 7, 9, 10, 11, 12, 13, 14, 15, 16]] == -1).all()


@pytest.mark.parametrize("A", [9, 82, 300, 9001])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_strides_offsets_and_untouched_neighbours(A, dtype):
    rng = np.random.default_rng(A + 5)
    B, pad = 7, 13
    for off in (0, 1, 3):
        big = torch.full((B, A + pad), float("nan"), dtype=TYPES[dtype], device="cuda")
        z = big[:, off : off + A]
        src, u, _ = inputs(rng, B, A, TYPES[dtype])
        z.copy_(src)
        lb = torch.zeros(B, A + pad, dtype=torch.uint8, device="cuda")
        legal = lb[:, 5 - off : 5 - off + A]
        legal.copy_(torch.from_numpy((rng.uniform(size=(B, A)) < 0.7).astype(np.uint8)))
        wide = torch.full((B + 2, A + pad), 7.0, device="cuda")
        out = dict(action=torch.full((B,), 77, dtype=torch.int32, device="cuda"), logprob=torch.empty(B, device="cuda"),
                   kept=torch.empty(B, dtype=torch.int32, device="cuda"), probs=wide[1 : B + 1, off : off + A])
        check(z, u, legal=legal, out=out, top_k=6, top_p=0.9)
        w = wide.clone()
        w[1 : B + 1, off : off + A] = 7.0
        assert (w == 7.0).all()
        one = z[2:3].expand(B, A)                     # every row the same logits: stride 0
        check(one, u, legal=legal, top_p=0.8)


def test_many_rows_twice_and_alone():
    """A row's result depends on nothing but the row: a batch, again, and its rows one by one."""
    rng = np.random.default_rng(6)
    for B, A, f in ((5000, 82, dict(top_k=20, top_p=0.9)), (300, 1500, dict(top_p=0.95)), (9, 60000, dict(top_p=0.97)),
                    (9, 60000, dict(top_k=1000, top_p=0.9))):
        z, u, legal = inputs(rng, B, A, torch.bfloat16, mask="legal")
        a = ops.sample_actions(z, u, legal=legal, probs=True, **f)
        b = ops.sample_actions(z, u, legal=legal, probs=True, **f)
        for k in a:
            assert torch.equal(a[k], b[k]), k
        for i in range(0, B, max(1, B // 7)):
            c = ops.sample_actions(z[i : i + 1], u[i : i + 1], legal=legal[i : i + 1], probs=True, **f)
            for k in a:
                assert torch.equal(a[k][i : i + 1], c[k]), (k, i)


def test_streams_and_graph_replays():
    rng = np.random.default_rng(7)
    for B, A, f in ((64, 82, dict(top_k=9, top_p=0.9)), (4, 30000, dict(top_p=0.9)), (3, 30000, dict(top_k=50))):
        z, u, legal = inputs(rng, B, A, torch.float16, mask="legal")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):
                ops.sample_actions(z, u, legal=legal, **f)
        torch.cuda.current_stream().wait_stream(s)
        g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g1):
            o1 = ops.sample_actions(z, u, legal=legal, **f)
        with torch.cuda.graph(g2):
            o2 = ops.sample_actions(z, u, legal=legal, temperature=0.5, **f)
        for step in range(4):
            nz, nu, nl = inputs(rng, B, A, torch.float16, mask="legal")
            z.copy_(nz)
            u.copy_(nu)
            legal.copy_(nl)
            g1.replay()
            g2.replay()
            e1, e2 = ops.sample_actions(z, u, legal=legal, **f), ops.sample_actions(z, u, legal=legal, temperature=0.5, **f)
            torch.cuda.synchronize()
            for k in e1:
                assert torch.equal(o1[k], e1[k]) and torch.equal(o2[k], e2[k]), (step, k)


def test_no_rows_and_refusals_on_the_device():
    z, u = torch.zeros(0, 9, device="cuda"), torch.zeros(0, dtype=torch.float64, device="cuda")
    assert ops.sample_actions(z, u)["action"].numel() == 0
    z, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, dtype=torch.float64, device="cuda")
    with pytest.raises(capi.MuZeroError, match="other operands"):
        ops.sample_actions(z, u.cpu())
    host = torch.zeros(2, 9)
    a = capi.SampleArgs(rows=2, actions=9, dtype=0, temperature=1.0, top_p=1.0, logits=host.data_ptr(), row_stride=9, u=u.data_ptr(),
                        action=torch.zeros(2, dtype=torch.int32, device="cuda").data_ptr())
    assert capi.lib().mz_sample_actions(capi.C.byref(a), None, 0, None) == -1
    assert b"logits is not device memory" in capi.lib().mz_last_error(None)
    a.logits = z.data_ptr() + 2
    assert capi.lib().mz_sample_actions(capi.C.byref(a), None, 0, None) == -1
    assert b"aligned" in capi.lib().mz_last_error(None)

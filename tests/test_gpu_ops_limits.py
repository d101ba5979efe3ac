"""-m gpu: the operators at the ends of what their documentation allows: offsets beyond 32 bits, the longest rows, overlapping
operands (refused), two calls at once, one stream's memory used on another, and arguments of the wrong kind."""
import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests import op_refs
from tests.test_gpu_adapter import check as check_adapter
from tests.test_gpu_adapter import make
from tests.test_gpu_sample import check as check_sample
from tests.test_gpu_sample import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,A,pitch", [(2100, 9, 2**21 + 3), (2100, 300, 2**21 + 3), (140, 9000, 2**25 + 8), (70, 20000, 2**26 + 1)])
def test_sample_rows_far_apart(B, A, pitch):
    """Row offsets pass 2^32 elements, of logits (2 bytes each) and, in the same buffer, flags; probs from row to row as far."""
    rng = np.random.default_rng(A)
    z, u, legal = inputs(rng, B, A, torch.bfloat16, mask="some")
    wide = torch.empty(B * pitch, dtype=torch.bfloat16, device="cuda").view(B, pitch)
    wide[:, 5 : A + 5] = z
    flags = torch.empty(B * pitch, dtype=torch.uint8, device="cuda").view(B, pitch)
    flags[:, 1 : A + 1] = legal
    for kw in (dict(), dict(top_k=20, top_p=0.9)):
        check_sample(wide[:, 5 : A + 5], u, legal=flags[:, 1 : A + 1], **kw)
    if B * pitch < 2**33 and A < 1000:
        probs = torch.empty(B * pitch, dtype=torch.float32, device="cuda").view(B, pitch)[:, 2 : A + 2]
        out = dict(action=torch.empty(B, dtype=torch.int32, device="cuda"), logprob=torch.empty(B, device="cuda"),
                   kept=torch.empty(B, dtype=torch.int32, device="cuda"), probs=probs)
        check_sample(wide[:, 5 : A + 5], u, legal=flags[:, 1 : A + 1], top_p=0.9, out=out)


@pytest.mark.parametrize("M,N,off", [(40, 50, 8), (2100, 30, 3), (2100, 300, 8), (2100, 700, 3), (2100, 2200, 8)])
def test_adapter_rows_far_apart(M, N, off):
    """x, weight and y are columns of the same wide rows, whose offsets pass 2^32 elements."""
    rng, K, pitch = np.random.default_rng(N), 72, 2**21
    if M == 40:
        pitch = 2**27
    s = make(rng, M, K, N, 8, 5, "bf16")
    wide = torch.empty(max(M, N) * pitch, dtype=torch.bfloat16, device="cuda").view(max(M, N), pitch)
    wide[:M, off : off + K] = s["x"]
    wide[:N, 200 + off : 200 + off + K] = s["weight"]
    s["x"], s["weight"] = wide[:M, off : off + K], wide[:N, 200 + off : 200 + off + K]
    check_adapter(s, "bf16", out=wide[:M, 400 + off : 400 + off + N])


@pytest.mark.parametrize("M", [3, 100, 1200])
def test_adapters_beyond_32_bits(M):
    """A and B of more than 2^32 elements; the last adapter and the first are used."""
    rng, K, N, r, n = np.random.default_rng(M), 8192, 8192, 128, 4100
    a = torch.empty(n, r, K, dtype=torch.bfloat16, device="cuda")
    b = torch.empty(n, N, r, dtype=torch.bfloat16, device="cuda")
    if M > 3:   # narrower products, A alone beyond 32 bits
        N = 200
        b = torch.empty(n, N, r, dtype=torch.bfloat16, device="cuda")
    s = make(rng, M, K, N, r, 2, "bf16", scale=False)
    a[0], a[n - 1], b[0], b[n - 1] = s["a"][0], s["a"][1], s["b"][0], s["b"][1]
    y = ops.adapter_linear(s["x"], s["weight"], a, b, torch.where(s["index"] == 1, n - 1, s["index"]), bias=s["bias"])
    assert torch.equal(y, check_adapter(s, "bf16")) or M > 64   # (many rows: the number of adapters chooses the way of the sum)
    want, size = op_refs.adapter(**s)
    tol = (2 * (K + r + 2) * 2.0**-24 + 2.0**-16) * size
    assert (np.abs(y.double().cpu().numpy() - want) <= tol + 2.0**-8 * (np.abs(want) + tol)).all()


def test_longest_rows():
    """262144 entries, all equal and all but one masked, for the three types; and one entry in a row of its own."""
    for t in (torch.float32, torch.bfloat16, torch.float16):
        z = torch.zeros(3, 262144, dtype=t, device="cuda")
        legal = torch.ones(3, 262144, dtype=torch.uint8, device="cuda")
        legal[1] = 0
        legal[1, 262143] = 1
        legal[2] = 0
        u = torch.tensor([1.0, 0.5, 0.5], dtype=torch.float64, device="cuda")
        for kw in (dict(), dict(top_p=0.5), dict(top_k=200000), dict(top_k=7), dict(min_p=1.0), dict(temperature=0.0)):
            check_sample(z, u, legal=legal, **kw)
        check_sample(z[:, :1], u)


def test_overlapping_operands_are_refused():
    rng = np.random.default_rng(0)
    z, u, _ = inputs(rng, 6, 300, torch.float32)
    new = lambda: dict(action=torch.empty(6, dtype=torch.int32, device="cuda"), logprob=torch.empty(6, device="cuda"))  # noqa: E731
    k = torch.full((6,), 3, dtype=torch.int32, device="cuda")
    for change, kw in ((dict(probs=z), {}), (dict(logprob=z.view(-1)[7:13]), {}), (dict(action=k), dict(top_k=k)),
                       (dict(kept=u.view(torch.int32)[:6]), {})):
        with pytest.raises(capi.MuZeroError, match="overlaps"):
            ops.sample_actions(z, u, out={**new(), **change}, **kw)
    both = new()
    both["kept"] = both["action"]
    with pytest.raises(capi.MuZeroError, match="overlaps"):
        ops.sample_actions(z, u, out=both)
    s = make(rng, 6, 64, 64, 4, 3, "bf16")
    for name in ("x", "weight", "a", "b", "bias"):
        flat = s[name].reshape(-1)
        y = torch.empty(6 * 64 + 64, dtype=torch.bfloat16, device="cuda")
        if flat.numel() >= 6 * 64:
            out = flat[-6 * 64 :].view(6, 64)
        else:   # the bias inside the result
            s["bias"] = y[70:134]
            out = y[: 6 * 64].view(6, 64)
        with pytest.raises(capi.MuZeroError, match="overlaps"):
            ops.adapter_linear(**s, out=out)
    # columns of the same wider rows lie side by side
    s = make(rng, 6, 64, 64, 4, 3, "bf16")
    wide = torch.zeros(6, 160, dtype=torch.bfloat16, device="cuda")
    wide[:, 80:144] = s["x"]
    s["x"] = wide[:, 80:144]
    check_adapter(s, "bf16", out=wide[:, :64])
    with pytest.raises(capi.MuZeroError, match="overlaps"):
        ops.adapter_linear(**s, out=wide[:, 20:84])
    with pytest.raises(capi.MuZeroError, match="overlaps"):
        ops.adapter_linear(**s, out=wide[:, 96:160])


def test_arguments_of_the_wrong_kind():
    rng = np.random.default_rng(1)
    z, u, _ = inputs(rng, 4, 20, torch.float32)
    for kw in (dict(top_k=None), dict(top_k=2.5), dict(top_k="3"), dict(temperature=None), dict(top_p="0.5"), dict(min_p=10**400),
               dict(top_k=-(2**40))):
        with pytest.raises(capi.MuZeroError):
            ops.sample_actions(z, u, **kw)
    check_sample(z, u, top_k=2**40)
    s = make(rng, 4, 64, 32, 4, 2, "fp32")
    for change in (dict(bias=1.0), dict(scale=2.0), dict(index=[0, 1, 0, 1]), dict(b=None)):
        with pytest.raises(capi.MuZeroError):
            ops.adapter_linear(**{**s, **change})
    with pytest.raises(capi.MuZeroError, match="gradient"):
        ops.adapter_linear(**s, out=torch.empty(4, 32, device="cuda", requires_grad=True))


def test_two_streams_with_long_rows():
    """Rows that several workgroups share, two calls in flight, each with a workspace of its own."""
    rng = np.random.default_rng(2)
    one, two = (inputs(rng, 5, 50000, torch.bfloat16) for _ in range(2))
    kw = dict(top_k=50, top_p=0.9)
    want = [ops.sample_actions(z, u, **kw) for z, u, _ in (one, two)]
    torch.cuda.synchronize()
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        got = []
        for side, (z, u, _) in zip(sides, (one, two)):
            with torch.cuda.stream(side):
                got.append(ops.sample_actions(z, u, **kw))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            for name in w:
                assert torch.equal(g[name], w[name])

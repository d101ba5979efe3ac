"""-m gpu: raw-policy moves through the C ABI (mz_play_policy): the network's logits, per-game adapters on the policy head, the
draw.  Given the logits, actions, counts and distributions follow the 64-bit restatement of the sampling; the logits are those of
mz_initial_inference, and with adapters those of the CPU network oracle within the bars its own tests use (2e-4 for fp32, the
error model's 20 * 0.9 * 2^-11 for fp16 operands), once for the shared projection and once for the adapter's term, whose weights
are of the same size."""
import json
import os
import subprocess

import numpy as np
import pytest
import torch

from muzero_amd import capi, netspec, ops
from oracle.net import NetOracle
from tests import op_refs

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BARS = {capi.PRECISION_FP32: 2e-4, capi.PRECISION_F16: 20 * 0.9 * 2.0**-11, capi.PRECISION_BF16: 8 * 20 * 0.9 * 2.0**-11}


def context(name, precision, B, pool=0):
    spec = netspec.SPECS[name]()
    w = netspec.random_weights(spec, seed=3, ln_jitter=0.1)
    cfg = capi.make_config(spec, 8, 4, 50, known_bounds=(-spec.value_scale, spec.value_scale), max_games=B, precision=precision, pool_slots=pool)
    ctx = capi.Context(cfg)
    ctx.load_weights(netspec.pack_blob(spec, w))
    ctx.set_action_cells(netspec.action_cells_board(spec))
    return spec, w, ctx


def positions(rng, spec, B):
    obs = (rng.uniform(size=(B, spec.obs_planes, spec.height, spec.width)) < 0.3).astype(np.float32)
    legal = (rng.uniform(size=(B, spec.action_space)) < 0.6).astype(np.uint8)
    legal[:, 0] = 1
    legal[B // 2] = 0
    return obs, legal, rng.uniform(size=B)


def adapters(rng, spec, n, rank):
    K, A = 2 * spec.hw, spec.action_space
    return ((rng.standard_normal((n, rank, K)) / np.sqrt(K)).astype(np.float32), (rng.standard_normal((n, A, rank)) / np.sqrt(rank)).astype(np.float32),
            rng.uniform(0.3, 1.0, n).astype(np.float32))


def check_draw(o, legal, u, **kw):
    want = op_refs.sample(torch.from_numpy(o["logits"]), torch.from_numpy(u), legal=torch.from_numpy(legal), **kw)
    np.testing.assert_array_equal(o["action"], want["action"])
    np.testing.assert_array_equal(o["kept"], want["kept"])
    np.testing.assert_allclose(o["logprob"], want["logprob"], rtol=2.0**-24 + 1e-12, atol=1e-11)
    np.testing.assert_allclose(o["playout_policy"], want["probs"], rtol=2.0**-24 + 1e-11, atol=2.0**-149)


@pytest.mark.parametrize("precision", list(BARS))
@pytest.mark.parametrize("name", ["tictactoe", "go9", "pegsolitair"])
def test_moves_without_adapters_draw_from_the_networks_logits(name, precision):
    rng = np.random.default_rng(0)
    B = 37
    spec, _, ctx = context(name, precision, B, pool=B)
    obs, legal, u = positions(rng, spec, B)
    logits, _, value = ctx.initial_inference(obs, np.arange(B))
    for kw in (dict(), dict(temperature=0.7, top_k=5, top_p=0.9, min_p=0.02), dict(temperature=0.0)):
        o = ctx.play_policy(B, obs, legal, u, **kw)
        np.testing.assert_array_equal(o["logits"], logits)
        np.testing.assert_array_equal(o["value"], value)
        assert o["action"][B // 2] == -1 and (o["playout_policy"][B // 2] == 0).all()
        check_draw(o, legal, u, **kw)
    ctx.close()


@pytest.mark.parametrize("precision", [capi.PRECISION_FP32, capi.PRECISION_F16])
@pytest.mark.parametrize("name,B,rank", [("tictactoe", 5, 3), ("go9", 64, 4), ("go9", 130, 16), ("pegsolitair", 70, 8)])
def test_moves_with_an_adapter_per_game(name, B, rank, precision):
    rng = np.random.default_rng(B)
    spec, w, ctx = context(name, precision, B)
    obs, legal, u = positions(rng, spec, B)
    n = 6
    a, b, scale = adapters(rng, spec, n, rank)
    index = rng.integers(-1, n, B).astype(np.int32)
    net = NetOracle(spec, w)
    with torch.no_grad():
        state = net.representation(torch.as_tensor(obs, dtype=net.dtype))
        f = torch.relu(net._ln(net._c1(state, "pred.p.conv"), "pred.p.ln")).reshape(B, -1).double().numpy()
    want, _ = op_refs.adapter(torch.from_numpy(f), torch.from_numpy(w["pred.p.fc.w"]), torch.from_numpy(a), torch.from_numpy(b),
                              torch.from_numpy(index), bias=torch.from_numpy(w["pred.p.fc.b"]), scale=torch.from_numpy(scale))
    ctx.load_policy_adapters(a, b, scale)
    o = ctx.play_policy(B, obs, legal, u, adapter=index, temperature=0.9, top_k=7, top_p=0.95)
    bar = 2 * BARS[precision]
    np.testing.assert_allclose(o["logits"], want, rtol=bar, atol=bar)
    check_draw(o, legal, u, temperature=0.9, top_k=7, top_p=0.95)
    # device arrays, a subset of the outputs
    t = lambda v: torch.from_numpy(v).cuda()  # noqa: E731
    out = dict(action=torch.zeros(B, dtype=torch.int32, device="cuda"), logits=torch.zeros(B, spec.action_space, device="cuda"))
    torch.cuda.synchronize()
    ctx.play_policy(B, t(obs), t(legal), t(u), adapter=t(index), temperature=0.9, top_k=7, top_p=0.95, outputs=out)
    np.testing.assert_array_equal(out["action"].cpu().numpy(), o["action"])
    np.testing.assert_array_equal(out["logits"].cpu().numpy(), o["logits"])
    # the adapters stay when weights come, go when they are taken away; smaller batches
    ctx.load_weights(netspec.pack_blob(spec, w))
    o2 = ctx.play_policy(B - 1, obs[:-1], legal[:-1], u[:-1], adapter=index[:-1], temperature=0.9, top_k=7, top_p=0.95)
    np.testing.assert_allclose(o2["logits"], want[:-1], rtol=bar, atol=bar)
    ctx.load_policy_adapters()
    with pytest.raises(capi.MuZeroError, match="no policy adapters"):
        ctx.play_policy(B, obs, legal, u, adapter=index)
    ctx.close()


def test_the_search_does_not_notice():
    rng = np.random.default_rng(5)
    B = 24
    spec, w, ctx = context("go9", capi.PRECISION_F16, B)
    obs, legal, u = positions(rng, spec, B)
    legal[B // 2, :3] = 1
    g = -np.log(-np.log(rng.uniform(size=(B, spec.action_space))))
    before = ctx.search_moves(B, obs, legal, gumbel=g)
    a, b, scale = adapters(rng, spec, 3, 4)
    ctx.load_policy_adapters(a, b, scale)
    ctx.play_policy(B, obs, legal, u, adapter=np.zeros(B, np.int32))
    after = ctx.search_moves(B, obs, legal, gumbel=g)
    for k in before:
        np.testing.assert_array_equal(before[k], after[k])
    ctx.close()


def test_refusals():
    rng = np.random.default_rng(6)
    spec, w, ctx = context("tictactoe", capi.PRECISION_FP32, 4)
    obs, legal, u = positions(rng, spec, 4)
    a, b, scale = adapters(rng, spec, 2, 3)
    ctx.load_policy_adapters(a, b)
    for kw, text in ((dict(adapter=np.array([0, 1, 2, 0], np.int32)), "out of range"), (dict(temperature=-1.0), "temperature"),
                     (dict(top_p=0.0), "top_p"), (dict(top_k=-1), "top_k"), (dict(min_p=2.0), "min_p")):
        with pytest.raises(capi.MuZeroError, match=text):
            ctx.play_policy(4, obs, legal, u, **kw)
    with pytest.raises(capi.MuZeroError, match="B out of range"):
        ctx.play_policy(5, np.repeat(obs, 2, 0), np.repeat(legal, 2, 0), np.repeat(u, 2))
    with pytest.raises(capi.MuZeroError, match="rank"):
        ctx._check(capi.lib().mz_load_policy_adapters(ctx._h, 2, 129, a.ctypes.data, b.ctypes.data, None))
    with pytest.raises(capi.MuZeroError, match="action_space"):
        ctx.load_policy_adapters(a, b[:, :-1])
    ctx.close()
    fresh = capi.Context(capi.make_config(spec, 8, 4, 50, max_games=4))
    with pytest.raises(capi.MuZeroError, match="weights not loaded"):
        fresh.play_policy(4, obs, legal, u)
    fresh.close()


def test_projection_and_draw_in_one_graph():
    """The two operators as a decode step uses them: logits of a batch with mixed adapters, a token of each row, captured once and
    replayed on changed inputs, against the eager calls and the 64-bit draw from the same logits."""
    rng = np.random.default_rng(7)
    for B, K, V in ((1, 256, 500), (20, 512, 20000), (90, 128, 300)):
        t = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda().bfloat16()  # noqa: E731
        x, W, a, b = t(B, K), t(V, K) / K**0.5, t(4, 8, K) / K**0.5, t(4, V, 8)
        index = torch.from_numpy(rng.integers(-1, 4, B).astype(np.int32)).cuda()
        u = torch.from_numpy(rng.uniform(size=B)).cuda()

        def step():
            logits = ops.adapter_linear(x, W, a, b, index, out_dtype=torch.float32)
            return logits, ops.sample_actions(logits, u, temperature=0.8, top_k=40, top_p=0.9, probs=True)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gl, go = step()
        for _ in range(3):
            x.copy_(t(B, K))
            u.copy_(torch.from_numpy(rng.uniform(size=B)))
            index.copy_(torch.from_numpy(rng.integers(-1, 4, B).astype(np.int32)))
            graph.replay()
            el, eo = step()
            torch.cuda.synchronize()
            assert torch.equal(gl, el)
            for k in eo:
                assert torch.equal(go[k], eo[k]), k
            want = op_refs.sample(gl, u, temperature=0.8, top_k=40, top_p=0.9)
            np.testing.assert_array_equal(go["action"].cpu().numpy(), want["action"])
            np.testing.assert_array_equal(go["kept"].cpu().numpy(), want["kept"])


def test_host_self_play_with_device_drawn_moves(tmp_path):
    """The host mirror's justInitialInferencePolicy play with PlayParameters.samplePolicy."""
    spec = netspec.spec_tictactoe()
    blob = tmp_path / "w.f32"
    netspec.pack_blob(spec, netspec.random_weights(spec, seed=1)).tofile(blob)
    exe = os.path.join(ROOT, "muzero_amd", "host", "bin", "selfplay_main")
    runs = [json.loads(subprocess.run([exe, str(blob), "100", "5", "HYBRID", "fp32", "policy"], check=True, capture_output=True, text=True, timeout=100).stdout)
            for _ in range(2)]
    r = runs[0]
    assert r["games"] == 100 and r["illegal_actions"] == 0 and r["bad_lengths"] == 0 and r["bad_policy_targets"] == 0 and r["not_done"] == 0
    assert r["simulations"] == 0 and runs[0] == runs[1]

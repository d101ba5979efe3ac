"""-m gpu: the operators of muzero_amd.ops have no gradients, and say so for every tensor that could ask for one."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from muzero_amd import capi, ops
from tests.test_gpu_adapter import check as check_adapter
from tests.test_gpu_adapter import make
from tests.test_gpu_sample import check as check_sample
from tests.test_gpu_sample import inputs

pytestmark = pytest.mark.gpu
SETTINGS = ("temperature", "top_p", "min_p")


def sample_arguments(rows=5, actions=20):
    z, u, _ = inputs(np.random.default_rng(0), rows, actions, torch.float32)
    per_row = {k: torch.full((rows,), v, dtype=torch.float64, device="cuda") for k, v in zip(SETTINGS, (0.9, 0.8, 0.01))}
    out = dict(action=torch.empty(rows, dtype=torch.int32, device="cuda"), logprob=torch.empty(rows, device="cuda"),
               probs=torch.empty(rows, actions, device="cuda"), kept=torch.empty(rows, dtype=torch.int32, device="cuda"))
    return dict(logits=z, u=u, **per_row), out


@pytest.mark.parametrize("name", ["logits", "u", *SETTINGS, "logprob", "probs"])
def test_sampling_refuses(name):
    given, out = sample_arguments()
    where = given if name in given else out
    where[name] = where[name].clone().requires_grad_()
    with pytest.raises(capi.MuZeroError, match="gradient"):
        ops.sample_actions(**given, out=out)
    with torch.no_grad():
        check_sample(given.pop("logits"), given.pop("u"), out=out, **given)


@pytest.mark.parametrize("name", ["x", "weight", "a", "b", "bias", "scale"])
def test_projection_refuses(name):
    s = make(np.random.default_rng(1), 6, 40, 24, 3, 2, "fp32")
    s[name] = s[name].clone().requires_grad_()
    with pytest.raises(capi.MuZeroError, match="gradient"):
        ops.adapter_linear(**s)
    with torch.no_grad():
        check_adapter({k: v.detach() for k, v in s.items()}, "fp32")
        ops.adapter_linear(**s)


def test_what_was_refused_with_a_gradient_is_refused_without():
    """Under no_grad a tensor that requires one still has to have the right layout."""
    given, _ = sample_arguments()
    with torch.no_grad():
        given["u"] = torch.rand(10, dtype=torch.float64, device="cuda", requires_grad=True)[::2]
        with pytest.raises(capi.MuZeroError, match="u: must be contiguous"):
            ops.sample_actions(**given)


@pytest.mark.parametrize("name", ["logits", "u", *SETTINGS, "logprob", "probs"])
def test_sampling_refuses_tangents(name):
    given, out = sample_arguments()
    where = given if name in given else out
    with forward_ad.dual_level():
        check_sample(given["logits"], given["u"], out=out, **{k: given[k] for k in SETTINGS})
        where[name] = forward_ad.make_dual(where[name], torch.ones_like(where[name]))
        for context in (torch.enable_grad, torch.no_grad):
            with context(), pytest.raises(capi.MuZeroError, match="tangent"):
                ops.sample_actions(**given, out=out)


@pytest.mark.parametrize("name", ["x", "weight", "a", "b", "bias", "scale"])
def test_projection_refuses_tangents(name):
    s = make(np.random.default_rng(2), 6, 40, 24, 3, 2, "fp32")
    with forward_ad.dual_level():
        check_adapter(s, "fp32")
        s[name] = forward_ad.make_dual(s[name], torch.ones_like(s[name]))
        with pytest.raises(capi.MuZeroError, match="tangent"):
            ops.adapter_linear(**s)


def test_derivatives_by_functions_end_in_an_error():
    given, _ = sample_arguments()
    s = make(np.random.default_rng(3), 6, 40, 24, 3, 2, "fp32")
    sample = lambda z: ops.sample_actions(**{**given, "logits": z})["logprob"]  # noqa: E731
    project = lambda x: ops.adapter_linear(**{**s, "x": x})  # noqa: E731
    for f, v in ((sample, given["logits"]), (project, s["x"])):
        with pytest.raises((capi.MuZeroError, RuntimeError)):
            torch.func.jvp(f, (v,), (torch.ones_like(v),))
        with pytest.raises((capi.MuZeroError, RuntimeError)):
            torch.func.grad(lambda t: f(t).sum())(v)
        with pytest.raises((capi.MuZeroError, RuntimeError)):
            torch.func.vmap(f)(v[None])


@pytest.mark.parametrize("name", ["logprob", "probs"])
def test_a_graph_notices_that_its_saved_sample_was_overwritten(name):
    given, out = sample_arguments()
    ops.sample_actions(**given, out=out)
    w = torch.ones_like(out[name], requires_grad=True)
    y = (w * out[name]).sum()
    ops.sample_actions(**given, out={k: v for k, v in out.items() if k != name})
    y.backward(retain_graph=True)
    ops.sample_actions(**given, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_graph_notices_that_its_saved_projection_was_overwritten():
    s = make(np.random.default_rng(4), 6, 40, 24, 3, 2, "fp32")
    out = ops.adapter_linear(**s)
    w = torch.ones_like(out, requires_grad=True)
    y = (w * out).sum()
    ops.adapter_linear(**s)
    y.backward(retain_graph=True)
    ops.adapter_linear(**s, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_outputs_made_in_inference_mode():
    s = make(np.random.default_rng(5), 6, 40, 24, 3, 2, "fp32")
    given, _ = sample_arguments()
    with torch.inference_mode():
        _, out = sample_arguments()
        ops.sample_actions(**given, out=out)
        y = torch.empty(6, 24, device="cuda")
        check_adapter(s, "fp32", out=y)
    with torch.no_grad():
        ops.sample_actions(**given, out=out)
        check_adapter(s, "fp32", out=y)

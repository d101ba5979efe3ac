"""CPU: what capi.Context hands to the C ABI, seen by a stand-in for the library that reads the arguments as the library would."""
import ctypes as C

import numpy as np
import pytest
import torch

from muzero_amd import capi, netspec


def read(p, dtype, n):
    p = getattr(p, "value", p)
    return np.frombuffer((C.c_char * (n * np.dtype(dtype).itemsize)).from_address(p), dtype).copy()


class Library:
    """Remembers what arrives, in the types and sizes of the header."""

    def __init__(self, B, spec):
        self.B, self.A, self.O = B, spec.action_space, spec.obs_planes * spec.hw

    def mz_destroy(self, h):
        pass

    def take_memory(self):
        """What the call allocates: memory that belongs to nobody when it begins gets other contents."""
        B, A = self.B, self.A
        self.taken = [np.full(n, 255, np.uint8) for n in (B, 4 * B, 8 * B, B * A, 4 * B * A, 8 * B * A, 4 * B * self.O) for _ in range(4)]

    def mz_play_policy(self, h, B, obs, legal, adapter, sampling, u, out):
        self.take_memory()
        self.sampling = sampling._obj
        self.got = dict(obs=read(obs, np.float32, self.B * self.O), legal=read(legal, np.uint8, self.B * self.A),
                        adapter=None if adapter is None else read(adapter, np.int32, self.B), u=read(u, np.float64, self.B))
        return 0

    def mz_search_moves(self, h, B, obs, legal, to_play, sims, gumbel, dirichlet, expl, u, out):
        self.take_memory()
        self.got = dict(obs=read(obs, np.float32, self.B * self.O), legal=read(legal, np.uint8, self.B * self.A),
                        to_play=read(to_play, np.uint8, self.B), num_simulations=read(sims, np.int32, self.B),
                        gumbel=read(gumbel, np.float64, self.B * self.A), u=read(u, np.float64, self.B))
        return 0


@pytest.fixture
def context(monkeypatch):
    spec, B = netspec.spec_tictactoe(), 6
    library = Library(B, spec)
    monkeypatch.setattr(capi, "lib", lambda: library)
    ctx = object.__new__(capi.Context)
    ctx.cfg = capi.make_config(spec, 8, 4, 50, max_games=B)
    ctx.A, ctx._h = spec.action_space, C.c_void_p()
    return ctx, library, spec, B


def converted(rng, spec, B):
    """Arguments of types that have to be converted first: the copies must live until the call returns."""
    return dict(obs=rng.integers(0, 2, (B, spec.obs_planes, spec.height, spec.width)).astype(np.float64),
                legal=rng.integers(0, 2, (B, spec.action_space)).astype(bool), u=rng.uniform(size=B).tolist())


def same(got, given):
    for k, v in given.items():
        np.testing.assert_array_equal(got[k], np.asarray(v).reshape(-1), err_msg=k)


def test_converted_arguments_of_play_policy(context):
    ctx, library, spec, B = context
    rng = np.random.default_rng(0)
    for _ in range(5):
        given = dict(converted(rng, spec, B), adapter=rng.integers(-1, 9, B))
        ctx.play_policy(B, **given)
        same(library.got, given)


def test_converted_arguments_of_search_moves(context):
    ctx, library, spec, B = context
    rng = np.random.default_rng(1)
    for _ in range(5):
        given = dict(converted(rng, spec, B), to_play=rng.integers(0, 2, B), num_simulations=rng.integers(1, 9, B),
                     gumbel=rng.uniform(size=(B, spec.action_space)).astype(np.float32))
        ctx.search_moves(B, **given)
        same(library.got, given)


def test_play_policy_keeps_top_k_whole(context):
    """A number beyond the field's 32 bits keeps all actions; it is not cut to its low bits (0: off, or 3 of them)."""
    ctx, library, spec, B = context
    given = converted(np.random.default_rng(2), spec, B)
    for k, arrives in ((5, 5), (2**32, 2**31 - 1), (2**32 + 3, 2**31 - 1), (2**40, 2**31 - 1), (-(2**32) + 3, -1), (np.int64(7), 7)):
        ctx.play_policy(B, **given, top_k=k)
        assert library.sampling.top_k == arrives


@pytest.mark.parametrize("change,text", [
    (dict(u=np.zeros(5)), "u: has 5 elements, needs 6"), (dict(u=torch.zeros(6)), "u: must be .* float64"),
    (dict(u=torch.zeros(12, dtype=torch.float64)[::2]), "u: must be contiguous"), (dict(legal=np.ones((5, 9), np.uint8)), "legal: has 45"),
    (dict(legal=torch.ones(6, 9)), "legal"), (dict(legal=np.full((6, 9), 256)), "legal: holds values"), (dict(obs=np.zeros((6, 3, 3))), "obs: has 54"),
    (dict(obs=torch.zeros(6, 300, dtype=torch.float16)), "obs"), (dict(adapter=np.full(6, 2**32)), "adapter: holds values"),
    (dict(adapter=np.full(6, 0.5)), "adapter: holds values"), (dict(adapter=torch.zeros(6, dtype=torch.int64)), "adapter"),
    (dict(adapter=[[0, 1], [2]]), "adapter"), (dict(u="0.5"), "u: a numpy array"), (dict(top_k=2.5), "must be numbers"),
    (dict(top_k=None), "must be numbers"), (dict(temperature=None), "must be numbers"), (dict(min_p="0"), "must be numbers"),
    (dict(outputs=dict(action=np.zeros(6, np.int64))), "action"), (dict(outputs=dict(logits=np.zeros((6, 8), np.float32))), "logits: has 48"),
    (dict(outputs=dict(value=torch.zeros(6))), "value"), (dict(outputs=dict(kept=[0] * 6)), "kept")])
def test_play_policy_refuses(context, change, text):
    ctx, library, spec, B = context
    with pytest.raises(capi.MuZeroError, match=text):
        ctx.play_policy(B, **{**converted(np.random.default_rng(3), spec, B), **change})


def test_play_policy_takes_more_than_it_needs_and_addresses(context):
    ctx, library, spec, B = context
    given = converted(np.random.default_rng(4), spec, B)
    u = torch.rand(9, dtype=torch.float64)
    given.update(u=u, legal=torch.ones(6, 9, dtype=torch.bool), adapter=torch.zeros(6, dtype=torch.int32))
    ctx.play_policy(B, **given)
    np.testing.assert_array_equal(library.got["u"], u[:6].numpy())
    ctx.play_policy(B, **{**given, "u": u.data_ptr()})
    np.testing.assert_array_equal(library.got["u"], u[:6].numpy())


@pytest.mark.parametrize("change", [dict(a=np.zeros((3, 18))), dict(b=None), dict(b=1.0), dict(a=[[1.0], [2.0, 3.0]]), dict(a=np.zeros((0, 2, 18))),
                                    dict(a=torch.zeros(3, 2, 18, dtype=torch.float64)), dict(a=torch.zeros(3, 18, 2).transpose(1, 2)),
                                    dict(scale=np.ones(2)), dict(scale=2.0), dict(scale="2")])
def test_load_policy_adapters_refuses(context, change):
    ctx = context[0]
    with pytest.raises(capi.MuZeroError):
        ctx.load_policy_adapters(**{**dict(a=np.zeros((3, 2, 18)), b=np.zeros((3, 9, 2))), **change})

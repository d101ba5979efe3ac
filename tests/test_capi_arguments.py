"""CPU: what capi.Context hands to the C ABI, seen by a stand-in for the library that reads the arguments as the library would."""
import ctypes as C

import numpy as np
import pytest

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

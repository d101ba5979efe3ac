"""CPU: what the operators of muzero_amd.ops / their C entries refuse, before anything could be queued, and struct layouts."""
import ctypes as C

import numpy as np
import pytest
import torch

from muzero_amd import capi, ops
from tests import op_refs


def last_error():
    return capi.lib().mz_last_error(None).decode()


def sample_args(**kw):
    a = capi.SampleArgs(rows=2, actions=9, dtype=0, temperature=1.0, top_p=1.0, row_stride=9, logits=64, u=64, action=64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(actions=0), "actions"), (dict(actions=262145), "actions"), (dict(dtype=3), "dtype"),
    (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(top_k=-1), "top_k"), (dict(top_p=0.0), "top_p"), (dict(top_p=1.01), "top_p"), (dict(top_p=float("nan")), "top_p"),
    (dict(min_p=-0.1), "min_p"), (dict(min_p=1.1), "min_p"), (dict(row_stride=-9), "strides"), (dict(legal=64, legal_stride=-1), "strides"),
    (dict(probs=64, probs_stride=8), "probs_stride"), (dict(logits=None), "NULL"), (dict(u=None), "NULL"), (dict(action=None), "NULL")])
def test_sample_refuses(change, text):
    a = sample_args(**change)
    assert capi.lib().mz_sample_actions(C.byref(a), None, 0, None) == -1
    assert text in last_error()
    assert capi.lib().mz_sample_workspace_bytes(C.byref(a)) == 0


def test_null_args_and_no_rows():
    assert capi.lib().mz_sample_actions(None, None, 0, None) == -1 and "NULL" in last_error()
    a = sample_args(rows=0, logits=None, u=None, action=None)
    assert capi.lib().mz_sample_actions(C.byref(a), None, 0, None) == 0


def test_host_memory_is_refused():
    z, u, act = np.zeros((2, 9), np.float32), np.zeros(2), np.zeros(2, np.int32)
    a = sample_args(logits=z.ctypes.data, u=u.ctypes.data, action=act.ctypes.data)
    assert capi.lib().mz_sample_actions(C.byref(a), None, 0, None) == -1
    assert "logits is not device memory" in last_error()
    with pytest.raises(capi.MuZeroError, match="GPU"):
        ops.sample_actions(torch.zeros(2, 9), torch.zeros(2, dtype=torch.float64))
    with pytest.raises(capi.MuZeroError, match="2-d"):
        ops.sample_actions(torch.zeros(9), torch.zeros(1, dtype=torch.float64))


def test_struct_layout():
    assert C.sizeof(capi.SampleArgs) == 4 * 4 + 3 * 8 + 14 * 8 == ops._SAMPLE.size
    assert C.sizeof(capi.AdapterArgs) == ops._ADAPTER.size
    a = capi.SampleArgs.from_buffer_copy(ops._SAMPLE.pack(*range(1, 5), 0.5, 0.25, 0.125, *range(11, 25)))
    assert (a.rows, a.top_k, a.temperature, a.min_p, a.logits, a.u, a.action, a.probs_stride) == (1, 4, 0.5, 0.125, 11, 15, 20, 24)


def test_the_restatement_on_a_row_done_by_hand():
    # weights 4, 2, 1, 1 (T = 1 / ln 2): ranks 2, 0, 1, 3
    z, ok, T = np.array([1.0, 0.0, 2.0, 0.0]), np.ones(4, bool), 1 / np.log(2)
    assert op_refs.sample_row(z, ok, T, 0, 1.0, 0.0, 0.0)[:1] == (0,)
    assert op_refs.sample_row(z, ok, T, 2, 1.0, 0.0, 0.4)[0] == 2           # 0.4 * 6 = 2.4 > 2
    assert op_refs.sample_row(z, ok, T, 0, 0.5001, 0.0, 0.3)[2] == 2        # 4 < 0.5001 * 8
    assert op_refs.sample_row(z, ok, T, 0, 0.49, 0.0, 0.3)[:1] == (2,)
    assert op_refs.sample_row(z, ok, T, 0, 1.0, 0.26, 0.9)[2] == 2
    assert op_refs.sample_row(z, np.zeros(4, bool), T, 0, 1.0, 0.0, 0.9)[0] == -1


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(in_features=0), "in_features"), (dict(out_features=0), "out_features"), (dict(rank=0), "rank"),
    (dict(rank=129), "rank"), (dict(adapters=0), "adapters"), (dict(dtype=3), "dtype"), (dict(out_dtype=2), "out_dtype"),
    (dict(x_stride=-1), "x_stride"), (dict(weight_stride=63), "weight_stride"), (dict(y_stride=31), "y_stride"), (dict(x=None), "NULL"),
    (dict(weight=None), "NULL"), (dict(a=None), "NULL"), (dict(b=None), "NULL"), (dict(index=None), "NULL"), (dict(y=None), "NULL")])
def test_adapter_refuses(change, text):
    a = capi.AdapterArgs(rows=2, in_features=64, out_features=32, rank=4, adapters=2, dtype=1, out_dtype=1, x=64, x_stride=64,
                         weight=64, weight_stride=64, a=64, b=64, index=64, y=64, y_stride=32)
    for k, v in change.items():
        setattr(a, k, v)
    assert capi.lib().mz_adapter_linear(C.byref(a), None, 0, None) == -1
    assert text in last_error()
    assert capi.lib().mz_adapter_workspace_bytes(C.byref(a)) == 0


def test_adapter_needs_device_tensors():
    z = torch.zeros
    assert C.sizeof(capi.AdapterArgs) == 8 * 4 + 12 * 8 - 8
    with pytest.raises(capi.MuZeroError, match="GPU"):
        ops.adapter_linear(z(2, 8), z(4, 8), z(1, 2, 8), z(1, 4, 2), z(2, dtype=torch.int32))


def test_adapter_of_no_rows():
    a = capi.AdapterArgs(rows=0, in_features=64, out_features=32, rank=4, adapters=2, dtype=1, out_dtype=1, x_stride=64,
                         weight_stride=64, y_stride=32)
    assert capi.lib().mz_adapter_workspace_bytes(C.byref(a)) == 0
    assert capi.lib().mz_adapter_linear(C.byref(a), None, 0, None) == 0


def test_policy_struct_layouts():
    assert C.sizeof(capi.PolicySampling) == 32 and C.sizeof(capi.PolicyOutputs) == 48


@pytest.mark.parametrize("change,text", [(dict(in_features=2**26 + 1, x_stride=2**26 + 1, weight_stride=2**26 + 1), "in_features"),
                                         (dict(rows=2**30), "too many"), (dict(rows=2**20, out_features=2**20, y_stride=2**20), "too many"),
                                         (dict(out_features=2**26 + 1, y_stride=2**26 + 1), "too many")])
def test_adapter_refuses_sizes_beyond_its_limits(change, text):
    a = capi.AdapterArgs(rows=2, in_features=64, out_features=32, rank=4, adapters=2, dtype=1, out_dtype=1, x=64, x_stride=64,
                         weight=64, weight_stride=64, a=64, b=64, index=64, y=64, y_stride=32)
    for k, v in change.items():
        setattr(a, k, v)
    assert capi.lib().mz_adapter_linear(C.byref(a), None, 0, None) == -1
    assert text in last_error()
    assert capi.lib().mz_adapter_workspace_bytes(C.byref(a)) == 0

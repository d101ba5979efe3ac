"""The library's operators on torch tensors (mz_sample_actions, mz_adapter_linear of include/muzero_hip.h): checks of types, shapes and
devices, then one call of the C ABI on torch's current stream of the tensors' device.  Nothing is copied, converted or
synchronised; a call can be captured into a torch.cuda.graph.  Errors are capi.MuZeroError."""
import torch

from . import capi

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # MZ_DTYPE_*


def _need(ok, text):
    if not ok:
        raise capi.MuZeroError(text)


def _tensor(t, name, dtype, shape, device, dense=True):
    """t as a tensor of that dtype, shape and device whose rows are contiguous (dense: entirely)."""
    _need(isinstance(t, torch.Tensor), f"{name}: a torch tensor is needed")
    _need(t.dtype == dtype, f"{name}: {t.dtype}, needs {dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name}: shape {tuple(t.shape)}, needs {tuple(shape)}")
    _need(t.device == device, f"{name}: on {t.device}, the other operands on {device}")
    if dense:
        _need(t.is_contiguous(), f"{name}: must be contiguous")
    else:
        _need(t.dim() < 1 or t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the last dimension must be contiguous")
    return t.data_ptr()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _finish(rc):
    if rc != 0:
        raise capi.MuZeroError(capi.lib().mz_last_error(None).decode())


def _workspace(need, given, device):
    """(tensor to keep alive, address, bytes).  torch's allocator hands the memory out per stream (and per graph)."""
    if given is not None:
        _need(given.dtype == torch.uint8 and given.is_contiguous() and given.device == device,
              f"workspace: a contiguous uint8 tensor on {device} is needed")
        return given, given.data_ptr(), given.numel()
    if need == 0:
        return None, None, 0
    w = torch.empty(need, dtype=torch.uint8, device=device)
    return w, w.data_ptr(), need


def sample_actions(logits, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=False, out=None,
                   workspace=None):
    """One action per row of `logits` [B, A] (float32, bfloat16 or float16), drawn with u [B] float64 in [0, 1] after
    temperature, top-k, top-p and min-p (mz_sample_actions has the definition).  `legal` [B, A] uint8 or bool; temperature,
    top_p, min_p: a number or a float64 tensor [B]; top_k: a number or an int32 tensor [B].

    Returns dict(action int32 [B], logprob float32 [B], kept int32 [B], and with probs=True probs float32 [B, A]).  `out`: such
    a dict of tensors to write into instead (action required, the others as wanted)."""
    _need(isinstance(logits, torch.Tensor) and logits.dim() == 2, "logits: a 2-d torch tensor is needed")
    _need(logits.is_cuda, "logits: must be on a GPU")
    _need(logits.dtype in DTYPES, f"logits: {logits.dtype} is not supported")
    B, A = logits.shape
    dev = logits.device
    a = capi.SampleArgs()
    a.rows, a.actions, a.dtype = B, A, DTYPES[logits.dtype]
    a.logits = _tensor(logits, "logits", logits.dtype, (B, A), dev, dense=False)
    a.row_stride = _row_stride(logits)
    if legal is not None:
        _need(isinstance(legal, torch.Tensor) and legal.dtype in (torch.uint8, torch.bool), "legal: uint8 or bool is needed")
        a.legal = _tensor(legal, "legal", legal.dtype, (B, A), dev, dense=False)
        a.legal_stride = _row_stride(legal)
    a.u = _tensor(u, "u", torch.float64, (B,), dev)
    if isinstance(temperature, torch.Tensor):
        a.row_temperature = _tensor(temperature, "temperature", torch.float64, (B,), dev)
    else:
        a.temperature = temperature
    if isinstance(top_k, torch.Tensor):
        a.row_top_k = _tensor(top_k, "top_k", torch.int32, (B,), dev)
    else:
        _need(0 <= top_k, "top_k must be >= 0")
        a.top_k = min(int(top_k), 2**31 - 1)
    if isinstance(top_p, torch.Tensor):
        a.row_top_p = _tensor(top_p, "top_p", torch.float64, (B,), dev)
    else:
        a.top_p = top_p
    if isinstance(min_p, torch.Tensor):
        a.row_min_p = _tensor(min_p, "min_p", torch.float64, (B,), dev)
    else:
        a.min_p = min_p
    if out is None:
        out = dict(action=torch.empty(B, dtype=torch.int32, device=dev), logprob=torch.empty(B, device=dev),
                   kept=torch.empty(B, dtype=torch.int32, device=dev))
        if probs:
            out["probs"] = torch.empty(B, A, device=dev)
    _need("action" in out, "out: 'action' is needed")
    a.action = _tensor(out["action"], "out['action']", torch.int32, (B,), dev)
    if out.get("logprob") is not None:
        a.logprob = _tensor(out["logprob"], "out['logprob']", torch.float32, (B,), dev)
    if out.get("kept") is not None:
        a.kept = _tensor(out["kept"], "out['kept']", torch.int32, (B,), dev)
    if out.get("probs") is not None:
        a.probs = _tensor(out["probs"], "out['probs']", torch.float32, (B, A), dev, dense=False)
        a.probs_stride = _row_stride(out["probs"])
    L = capi.lib()
    ref = capi.C.byref(a)
    keep, ws, nbytes = _workspace(L.mz_sample_workspace_bytes(ref), workspace, dev)
    _finish(L.mz_sample_actions(ref, ws, nbytes, torch.cuda.current_stream(dev).cuda_stream))
    return out


def adapter_linear(x, weight, a, b, index, bias=None, scale=None, out_dtype=None, out=None, workspace=None):
    """x [M, K] @ weight [N, K]^T + bias [N], plus each row's own adapter i = index[m] (int32 [M], -1 = none):
    scale[i] * (x[m] @ a[i]^T) @ b[i]^T with a [n, r, K], b [n, N, r] and scale float32 [n] (None: 1).  All of one type (float32,
    bfloat16, float16); the result [M, N] has it too, or float32 with out_dtype=torch.float32 (mz_adapter_linear)."""
    _need(isinstance(x, torch.Tensor) and x.dim() == 2, "x: a 2-d torch tensor is needed")
    _need(x.is_cuda, "x: must be on a GPU")
    t, dev = x.dtype, x.device
    _need(t in DTYPES, f"x: {t} is not supported")
    M, K = x.shape
    _need(isinstance(weight, torch.Tensor) and weight.dim() == 2, "weight: a 2-d torch tensor is needed")
    _need(isinstance(a, torch.Tensor) and a.dim() == 3, "a: a 3-d torch tensor is needed")
    N, (n, r, _) = weight.shape[0], a.shape
    if out_dtype is None:
        out_dtype = t if out is None else out.dtype
    _need(out_dtype in DTYPES, f"out_dtype: {out_dtype} is not supported")
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=dev)
    g = capi.AdapterArgs()
    g.rows, g.in_features, g.out_features, g.rank, g.adapters = M, K, N, r, n
    g.dtype, g.out_dtype = DTYPES[t], DTYPES[out_dtype]
    g.x = _tensor(x, "x", t, (M, K), dev, dense=False)
    g.x_stride = _row_stride(x)
    g.weight = _tensor(weight, "weight", t, (N, K), dev, dense=False)
    g.weight_stride = _row_stride(weight)
    if bias is not None:
        g.bias = _tensor(bias, "bias", t, (N,), dev)
    g.a = _tensor(a, "a", t, (n, r, K), dev)
    g.b = _tensor(b, "b", t, (n, N, r), dev)
    if scale is not None:
        g.scale = _tensor(scale, "scale", torch.float32, (n,), dev)
    g.index = _tensor(index, "index", torch.int32, (M,), dev)
    g.y = _tensor(out, "out", out_dtype, (M, N), dev, dense=False)
    g.y_stride = _row_stride(out)
    L = capi.lib()
    ref = capi.C.byref(g)
    keep, ws, nbytes = _workspace(L.mz_adapter_workspace_bytes(ref), workspace, dev)
    _finish(L.mz_adapter_linear(ref, ws, nbytes, torch.cuda.current_stream(dev).cuda_stream))
    return out

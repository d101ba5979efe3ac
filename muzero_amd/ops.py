"""The library's operators on torch tensors (mz_sample_actions, mz_adapter_linear of include/muzero_hip.h): checks of types, shapes and
devices, then one call of the C ABI on torch's current stream of the tensors' device.  Nothing is copied, converted or
synchronised; a call can be captured into a torch.cuda.graph.  There are no gradients: inputs that ask for them are refused
while torch's grad mode is on, forward-mode tangents always.  Errors are capi.MuZeroError."""
import ctypes as C
import struct

import torch
from torch.autograd import forward_ad

from . import capi

# of a list of tensors, without the tests around it
_increment_version = getattr(torch._C, "_increment_version", None) or torch.autograd.graph.increment_version
# torch's current stream of a GPU, as a hipStream_t: the same number without a Stream object around it, where torch has that
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)
# the argument structs of the C ABI as bytes (capi.SampleArgs, capi.AdapterArgs have the fields): packing costs a quarter of
# filling a ctypes Structure, and these calls are short
_SAMPLE = struct.Struct("=4i3d14q")
_ADAPTER = struct.Struct("=8i11q")
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}   # MZ_DTYPE_*
_NUMBERS = (float, int)   # (a test for Tensor goes through its metaclass and is slow)
_entries = None


def _lib():
    """The operators' C entries, with the structs as bytes."""
    global _entries
    if _entries is None:
        capi.lib()   # fails loudly if the library is missing
        L = C.CDLL(capi.LIB_PATH)
        for name in ("mz_sample", "mz_adapter"):
            f = getattr(L, name + "_workspace_bytes")
            f.argtypes, f.restype = [C.c_char_p], C.c_size_t
        for name in ("mz_sample_actions", "mz_adapter_linear"):
            getattr(L, name).argtypes = [C.c_char_p, C.c_void_p, C.c_size_t, C.c_void_p]
        _entries = L
    return _entries


def _need(ok, text):
    if not ok:
        raise capi.MuZeroError(text)


def _tensor(t, name, dtype, shape, device, dense=True):
    """Address of t, a tensor of that dtype and shape on GPU `device` whose rows are contiguous (dense: all of it)."""
    try:   # one test for the usual case; which one failed is found out below
        if (t.dtype is dtype and t.shape == shape and t.get_device() == device and not t.requires_grad
                and (t.is_contiguous() or not dense and t.stride(-1) == 1)):
            return t.data_ptr()
    except AttributeError:
        pass
    _need(isinstance(t, torch.Tensor), f"{name}: a torch tensor is needed")
    _need(t.dtype == dtype, f"{name}: {t.dtype}, needs {dtype}")
    _need(tuple(t.shape) == tuple(shape), f"{name}: shape {tuple(t.shape)}, needs {tuple(shape)}")
    _need(t.get_device() == device, f"{name}: on {t.device}, the other operands on cuda:{device}")
    _need(t.is_contiguous() or not dense, f"{name}: must be contiguous")
    _need(t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name}: the last dimension must be contiguous")
    _need(not (t.requires_grad and torch.is_grad_enabled()),
          f"{name}: requires a gradient and this operator has none: call it under torch.no_grad()")
    return t.data_ptr()


def _row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _no_tangent(*values):
    for v in values:
        if isinstance(v, torch.Tensor) and v.is_floating_point() and forward_ad.unpack_dual(v).tangent is not None:
            raise capi.MuZeroError("an argument carries a forward-mode tangent and this operator has no derivative")


def _fail():
    raise capi.MuZeroError(capi.lib().mz_last_error(None).decode())


def _workspace(need, given, device):
    """(tensor to keep alive, address, bytes).  torch's allocator hands the memory out per stream (and per graph)."""
    if given is None and need == 0:
        return None, None, 0
    if given is not None:
        _need(isinstance(given, torch.Tensor) and given.dtype == torch.uint8 and given.is_contiguous() and given.get_device() == device,
              f"workspace: a contiguous uint8 tensor on cuda:{device} is needed")
        return given, given.data_ptr(), given.numel()
    w = torch.empty(need, dtype=torch.uint8, device=f"cuda:{device}")
    return w, w.data_ptr(), need


def sample_actions(logits, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, probs=False, out=None,
                   workspace=None):
    """One action per row of `logits` [B, A] (float32, bfloat16 or float16), drawn with u [B] float64 in [0, 1] after
    temperature, top-k, top-p and min-p (mz_sample_actions has the definition).  `legal` [B, A] uint8 or bool; temperature,
    top_p, min_p: a number or a float64 tensor [B]; top_k: a number or an int32 tensor [B].

    Returns dict(action int32 [B], logprob float32 [B], kept int32 [B], and with probs=True probs float32 [B, A]).  `out`: such
    a dict of tensors to write into instead (action required, the others as wanted)."""
    if not (isinstance(logits, torch.Tensor) and logits.dim() == 2):
        raise capi.MuZeroError("logits: a 2-d torch tensor is needed")
    t, dev = logits.dtype, logits.get_device()
    if dev < 0 or t not in DTYPES:
        raise capi.MuZeroError(f"logits: must be on a GPU and float32, bfloat16 or float16, not {t} on {logits.device}")
    if forward_ad._current_level >= 0:   # inside a dual_level
        _no_tangent(logits, u, temperature, top_p, min_p, *(out or {}).values())
    shape = logits.shape
    B, A = shape
    rows = (B,)
    p_legal, s_legal = 0, 0
    if legal is not None:
        lt = getattr(legal, "dtype", None)
        if lt is not torch.uint8 and lt is not torch.bool:
            raise capi.MuZeroError("legal: a uint8 or bool tensor is needed")
        p_legal, s_legal = _tensor(legal, "legal", lt, shape, dev, dense=False), _row_stride(legal)
    p_t = p_k = p_p = p_m = 0   # a number, or a tensor with one per row
    if type(temperature) not in _NUMBERS and isinstance(temperature, torch.Tensor):
        p_t, temperature = _tensor(temperature, "temperature", torch.float64, rows, dev), 0
    if type(top_k) not in _NUMBERS and isinstance(top_k, torch.Tensor):
        p_k, top_k = _tensor(top_k, "top_k", torch.int32, rows, dev), 0
    if type(top_p) not in _NUMBERS and isinstance(top_p, torch.Tensor):
        p_p, top_p = _tensor(top_p, "top_p", torch.float64, rows, dev), 0
    if type(min_p) not in _NUMBERS and isinstance(min_p, torch.Tensor):
        p_m, min_p = _tensor(min_p, "min_p", torch.float64, rows, dev), 0
    if type(top_k) is int and top_k >= 2**31:
        top_k = 2**31 - 1
    given = out is not None
    if not given:
        on = logits.device
        out = dict(action=torch.empty(B, dtype=torch.int32, device=on), logprob=torch.empty(B, dtype=torch.float32, device=on),
                   kept=torch.empty(B, dtype=torch.int32, device=on))
        if probs:
            out["probs"] = torch.empty(B, A, dtype=torch.float32, device=on)
    action, logprob, kept, probs = out.get("action"), out.get("logprob"), out.get("kept"), out.get("probs")
    p_action, p_logprob, p_kept, p_probs, s_probs = _tensor(action, "out['action']", torch.int32, rows, dev), 0, 0, 0, 0
    written = [action]
    if logprob is not None:
        p_logprob = _tensor(logprob, "out['logprob']", torch.float32, rows, dev)
        written.append(logprob)
    if kept is not None:
        p_kept = _tensor(kept, "out['kept']", torch.int32, rows, dev)
        written.append(kept)
    if probs is not None:
        p_probs, s_probs = _tensor(probs, "out['probs']", torch.float32, shape, dev, dense=False), _row_stride(probs)
        written.append(probs)
    p_logits, p_u = _tensor(logits, "logits", t, shape, dev, dense=False), _tensor(u, "u", torch.float64, rows, dev)
    try:
        args = _SAMPLE.pack(B, A, DTYPES[t], top_k, temperature, top_p, min_p, p_logits, _row_stride(logits), p_legal, s_legal, p_u,
                            p_t, p_k, p_p, p_m, p_action, p_logprob, p_kept, p_probs, s_probs)
    except (struct.error, OverflowError, TypeError) as e:
        raise capi.MuZeroError(f"sizes, temperature, top_k, top_p and min_p must be numbers in range ({e})") from None
    L = _entries or _lib()
    keep, ws, nbytes = _workspace(L.mz_sample_workspace_bytes(args), workspace, dev)
    if L.mz_sample_actions(args, ws, nbytes, _stream(dev)) != 0:
        _fail()
    if given:   # a graph that saved one of them must notice
        _increment_version(written)
    return out


def adapter_linear(x, weight, a, b, index, bias=None, scale=None, out_dtype=None, out=None, workspace=None):
    """x [M, K] @ weight [N, K]^T + bias [N], plus each row's own adapter i = index[m] (int32 [M], -1 = none):
    scale[i] * (x[m] @ a[i]^T) @ b[i]^T with a [n, r, K], b [n, N, r] and scale float32 [n] (None: 1).  All of one type (float32,
    bfloat16, float16); the result [M, N] has it too, or float32 with out_dtype=torch.float32 (mz_adapter_linear)."""
    for v, name, dims in ((x, "x", 2), (weight, "weight", 2), (a, "a", 3)):
        if not (isinstance(v, torch.Tensor) and v.dim() == dims):
            raise capi.MuZeroError(f"{name}: a {dims}-d torch tensor is needed")
    t, dev = x.dtype, x.get_device()
    if dev < 0 or t not in DTYPES:
        raise capi.MuZeroError(f"x: must be on a GPU and float32, bfloat16 or float16, not {t} on {x.device}")
    M, K = x.shape
    n, r, _ = a.shape
    N = weight.shape[0]
    given = out is not None
    if not given:
        out = torch.empty(M, N, dtype=t if out_dtype is None else out_dtype, device=x.device)
    elif out_dtype is None:
        out_dtype = getattr(out, "dtype", None)
    if out_dtype is None:
        out_dtype = t
    if out_dtype not in DTYPES:
        raise capi.MuZeroError(f"out: {out_dtype} is not supported")
    if forward_ad._current_level >= 0:   # inside a dual_level
        _no_tangent(x, weight, a, b, bias, scale, out)
    try:
        args = _ADAPTER.pack(
            M, K, N, r, n, DTYPES[t], DTYPES[out_dtype], 0,
            _tensor(x, "x", t, (M, K), dev, dense=False), _row_stride(x),
            _tensor(weight, "weight", t, (N, K), dev, dense=False), _row_stride(weight),
            0 if bias is None else _tensor(bias, "bias", t, (N,), dev),
            _tensor(a, "a", t, (n, r, K), dev), _tensor(b, "b", t, (n, N, r), dev),
            0 if scale is None else _tensor(scale, "scale", torch.float32, (n,), dev),
            _tensor(index, "index", torch.int32, (M,), dev), _tensor(out, "out", out_dtype, (M, N), dev, dense=False),
            _row_stride(out))
    except struct.error as e:
        raise capi.MuZeroError(f"sizes must be below 2^31 ({e})") from None
    L = _entries or _lib()
    keep, ws, nbytes = _workspace(L.mz_adapter_workspace_bytes(args), workspace, dev)
    if L.mz_adapter_linear(args, ws, nbytes, _stream(dev)) != 0:
        _fail()
    if given:   # a graph that saved it must notice
        _increment_version([out])
    return out

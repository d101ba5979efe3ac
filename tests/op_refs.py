"""Plain 64-bit restatements of the operators of muzero_amd.ops (test oracles, numpy on the host)."""
import math

import numpy as np
import torch


def bf16_round(x):
    return torch.as_tensor(x).to(torch.bfloat16)


def sample_row(z, ok, T, k, p, m, u):
    """(action, logprob, kept, probs) of one row: z float64 [A], ok bool [A] (legal, not NaN, not -inf)."""
    A = len(z)
    probs = np.zeros(A)
    ids = np.flatnonzero(ok)
    valid = (0 <= T < math.inf) and k >= 0 and 0 < p <= 1 and 0 <= m <= 1 and 0 <= u <= 1
    if not len(ids) or not valid:
        return -1, 0.0, 0, probs
    v = z[ids]
    if T == 0:
        a = ids[int(np.argmax(v))]
        probs[a] = 1.0
        return int(a), 0.0, 1, probs
    ranked = np.argsort(-v, kind="stable")
    top = v[ranked[0]]
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(v[ranked] == top, 0.0, (v[ranked] - top) / T)
    w = np.exp(x)
    n = min(k, len(ids)) if k > 0 else len(ids)
    if p < 1:
        s = np.cumsum(w[:n])
        n = int(np.sum(np.concatenate([[0.0], s[:-1]]) < p * s[-1]))
    if m > 0:
        n = min(n, int(np.sum(w[:n] >= m)))
    n = max(n, 1)
    order = np.argsort(ranked[:n])                      # the kept, in index order
    c = np.cumsum(w[:n][order])
    hit = np.flatnonzero((c > u * c[-1]) & (w[:n][order] > 0))
    j = int(hit[0]) if len(hit) else int(np.flatnonzero(w[:n][order])[-1])
    probs[ids[ranked[:n][order]]] = w[:n][order] / c[-1]
    return int(ids[ranked[:n][order][j]]), float(x[:n][order][j] - math.log(c[-1])), n, probs


def sample(logits, u, legal=None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    z = logits.float().cpu().numpy().astype(np.float64)
    ok = ~np.isnan(z) & (z != -np.inf)
    if legal is not None:
        ok &= legal.cpu().numpy() != 0
    u = u.cpu().numpy()
    par = [v.cpu().numpy() if isinstance(v, torch.Tensor) else np.full(len(z), v) for v in (temperature, top_k, top_p, min_p)]
    rows = [sample_row(z[i], ok[i], *(q[i] for q in par), u[i]) for i in range(len(z))]
    return dict(action=np.array([r[0] for r in rows], np.int32), logprob=np.array([r[1] for r in rows]),
                kept=np.array([r[2] for r in rows], np.int32), probs=np.array([r[3] for r in rows]))


def adapter(x, weight, a, b, index, bias=None, scale=None):
    """(y, size) in 64 bits on the host: y of mz_adapter_linear, and the sum of the absolute values of all terms of each y,
    which is what rounding errors of the sums go by."""
    f = lambda v: v.detach().cpu().double().numpy()  # noqa: E731
    x, w, a, b, index = f(x), f(weight), f(a), f(b), index.cpu().numpy()
    with np.errstate(invalid="ignore", over="ignore"):
        y, size = x @ w.T, np.abs(x) @ np.abs(w).T
        if bias is not None:
            y = y + f(bias)
            size = size + np.abs(f(bias))
        for i in np.unique(index):
            rows = np.flatnonzero(index == i)
            if i < -1 or i >= len(a):
                y[rows] = np.nan
            elif i >= 0:
                s = 1.0 if scale is None else float(scale[i])
                y[rows] += s * (x[rows] @ a[i].T) @ b[i].T
                size[rows] += abs(s) * (np.abs(x[rows]) @ np.abs(a[i]).T) @ np.abs(b[i]).T
    return y, size

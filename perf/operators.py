"""The language-model operators of this library, as a user's program calls them, next to their plain forms.

Two operators, which follow one another when a batch of requests (games, sequences) is answered from a network's last features:

  adapter_linear   y = x W^T + bias + scale[i] (x A[i]^T) B[i]^T, i = the row's own adapter: one shared projection with low-rank
                   adapters of many requests beside it
  sample_actions   an entry of each row of logits, drawn from a given random number after temperature, top-k, top-p and min-p

`listed()` / `draw(rng)` give cases, `prepare(case, seed)` makes what a program holds before the call, `run(state)` is one call:
of the library where `own` is set, of elementary torch operations otherwise.  `exact(case, seed)` is the definition in 64 bits.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- cases -------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one TicTacToe position answered by the raw policy: nothing but latency
        dict(name="sample_board3_one", op="sample", rows=1, actions=9, dtype="fp32", mask="legal", temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0, spread=1.5, probs=True, per_row=False),
        # every Go 9x9 game of a self-play batch plays one raw-policy move; the playout policy goes to the replay buffer; each
        # game has its own temperature and filters, and finished games have no legal move
        dict(name="sample_go9_batch", op="sample", rows=16384, actions=82, dtype="fp32", mask="some_empty", temperature=1.0,
             top_k=20, top_p=0.95, min_p=0.01, spread=2.0, probs=True, per_row=True),
        # PegSolitair's 196 actions, 16-bit logits as the MFMA networks hold them
        dict(name="sample_peg_batch", op="sample", rows=4096, actions=196, dtype="fp16", mask="legal", temperature=0.7, top_k=0,
             top_p=0.9, min_p=0.0, spread=2.0, probs=False, per_row=False),
        # one token of one sequence over a large vocabulary
        dict(name="sample_vocab_one", op="sample", rows=1, actions=131072, dtype="bf16", mask="none", temperature=0.8, top_k=50,
             top_p=0.9, min_p=0.0, spread=3.0, probs=False, per_row=False),
        # a decode batch, odd vocabulary, each sequence with its own settings
        dict(name="sample_vocab_64", op="sample", rows=64, actions=50257, dtype="fp32", mask="none", temperature=0.8, top_k=40,
             top_p=0.95, min_p=0.02, spread=3.0, probs=False, per_row=True),
        # the largest: a nucleus of tens of thousands of entries in flat 16-bit rows, no top-k to cut it short
        dict(name="sample_vocab_256_flat", op="sample", rows=256, actions=131072, dtype="bf16", mask="none", temperature=1.3,
             top_k=0, top_p=0.95, min_p=0.0, spread=2.0, probs=False, per_row=False),
        # the policy head of Go 9x9 (2 * 81 features, 82 actions) for one game with its own adapter
        dict(name="adapter_go9_head_one", op="adapter", rows=1, inner=162, outer=82, rank=4, adapters=4, dtype="fp32", bias=True,
             bare=0.0, order="mixed"),
        # the same for a whole batch: a population of 32 players shares one network
        dict(name="adapter_go9_head_batch", op="adapter", rows=16384, inner=162, outer=82, rank=8, adapters=32, dtype="fp32",
             bias=True, bare=0.1, order="mixed"),
        # one token through a projection
        dict(name="adapter_decode_one", op="adapter", rows=1, inner=4096, outer=4096, rank=16, adapters=8, dtype="bf16",
             bias=False, bare=0.0, order="mixed"),
        # a decode batch in which every sequence has an adapter of its own
        dict(name="adapter_decode_48", op="adapter", rows=48, inner=4096, outer=11000, rank=32, adapters=48, dtype="fp16",
             bias=False, bare=0.1, order="distinct"),
        # ragged prompt tokens of a few requests, nothing a multiple of a tile
        dict(name="adapter_ragged_1000", op="adapter", rows=1000, inner=2050, outer=1999, rank=12, adapters=5, dtype="bf16",
             bias=True, bare=0.2, order="runs"),
        # the largest: prompts of many requests in one batch
        dict(name="adapter_prompt_8192", op="adapter", rows=8192, inner=4096, outer=4096, rank=16, adapters=24, dtype="bf16",
             bias=False, bare=0.05, order="runs"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    if rng.random() < 0.5:
        actions = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 1, max(1, min(16384, 256 * 131072 // actions)))
        f = rng.randrange(5)
        return dict(op="sample", rows=rows, actions=actions, dtype=rng.choice(["fp32", "bf16", "fp16"]),
                    mask=rng.choice(["none", "legal", "some_empty"]), temperature=round(rng.uniform(0.3, 2.0), 3),
                    top_k=_log_int(rng, 1, actions) if f in (0, 1, 2) else 0,
                    top_p=round(rng.uniform(0.5, 0.999), 4) if f in (1, 2, 3) else 1.0,
                    min_p=round(rng.uniform(0.001, 0.2), 4) if f in (2, 4) else 0.0, spread=round(rng.uniform(0.5, 4.0), 3),
                    probs=rng.random() < 0.3, per_row=rng.random() < 0.5)
    inner, outer = _log_int(rng, 16, 8192), _log_int(rng, 8, 12000)
    rows = _log_int(rng, 1, max(1, min(16384, 8192 * 4096 * 4096 // (inner * outer))))
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if dtype == "fp32":
        rows = max(1, min(rows, 1024 * 4096 * 4096 // (inner * outer)))
    rank, adapters = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
    return dict(op="adapter", rows=rows, inner=inner, outer=outer, rank=rank, adapters=adapters, dtype=dtype,
                bias=rng.random() < 0.5, bare=rng.choice([0.0, 0.1, 0.5]), order=rng.choice(["mixed", "runs", "distinct"]))


# ---- inputs ------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(1000003 * seed + 17)
    dev = dict(device="cuda")
    t = TYPES[case["dtype"]]
    B = case["rows"]
    if case["op"] == "sample":
        A = case["actions"]
        # logits as a trained head gives them: a bell of `spread`, a few entries well above it
        logits = case["spread"] * torch.randn(B, A, generator=g, **dev)
        logits[torch.rand(B, A, generator=g, **dev) < 8.0 / (A + 8.0)] += 2.0 * case["spread"]
        logits = logits.to(t)
        legal = None
        if case["mask"] != "none":
            legal = torch.rand(B, A, generator=g, **dev) < 0.6
            legal[torch.arange(B, **dev), torch.randint(0, A, (B,), generator=g, **dev)] = True
            if case["mask"] == "some_empty":
                legal[torch.rand(B, generator=g, **dev) < 0.02] = False
            # what a masked place holds is nobody's business
            logits[~legal & (torch.rand(B, A, generator=g, **dev) < 0.05)] = float("nan")
            legal = legal.to(torch.uint8)
        T, k, p, m = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        if case["per_row"]:
            f64 = dict(dtype=torch.float64, generator=g, **dev)
            T = T * (0.5 + torch.rand(B, **f64))
            T[torch.rand(B, generator=g, **dev) < 0.05] = 0.0          # some rows play greedily
            if k:
                k = torch.randint(1, 2 * k + 1, (B,), generator=g, **dev).to(torch.int32)
            if p < 1.0:
                p = 1.0 - (1.0 - p) * 2.0 * torch.rand(B, **f64)
            if m:
                m = m * 2.0 * torch.rand(B, **f64)
        u = torch.rand(B, dtype=torch.float64, generator=g, **dev)
        out = dict(action=torch.empty(B, dtype=torch.int32, **dev), logprob=torch.empty(B, **dev),
                   kept=torch.empty(B, dtype=torch.int32, **dev))
        if case["probs"]:
            out["probs"] = torch.empty(B, A, **dev)
        return dict(op="sample", logits=logits, legal=legal, u=u, temperature=T, top_k=k, top_p=p, min_p=m, out=out)
    K, N, r, n = case["inner"], case["outer"], case["rank"], case["adapters"]
    x = torch.randn(B, K, generator=g, **dev).to(t)
    W = (torch.randn(N, K, generator=g, **dev) / math.sqrt(K)).to(t)
    bias = (0.1 * torch.randn(N, generator=g, **dev)).to(t) if case["bias"] else None
    a = (torch.randn(n, r, K, generator=g, **dev) / math.sqrt(K)).to(t)
    b = (torch.randn(n, N, r, generator=g, **dev) / math.sqrt(r)).to(t)
    scale = 0.25 + 0.5 * torch.rand(n, generator=g, **dev)
    if case["order"] == "distinct":
        index = torch.arange(B, **dev) % n
    else:
        index = torch.randint(0, n, (B,), generator=g, **dev)
        if case["order"] == "runs":       # the tokens of one request stand together
            index = index[torch.sort(torch.randint(0, 4 * n, (B,), generator=g, **dev)).values % B]
    index[torch.rand(B, generator=g, **dev) < case["bare"]] = -1
    return dict(op="adapter", x=x, weight=W, bias=bias, a=a, b=b, scale=scale, index=index.to(torch.int32),
                out=torch.empty(B, N, dtype=t, **dev))


# ---- one call ----------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        from muzero_amd import ops
        s = state
        if s["op"] == "sample":
            return ops.sample_actions(s["logits"], s["u"], legal=s["legal"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"], out=s["out"])
        return dict(y=ops.adapter_linear(s["x"], s["weight"], s["a"], s["b"], s["index"], bias=s["bias"], scale=s["scale"],
                                         out=s["out"]))
    return _plain_sample(state) if state["op"] == "sample" else dict(y=_plain_adapter(state))


def _column(v):
    return v[:, None] if isinstance(v, torch.Tensor) else v


def _plain_sample(s):
    logits, legal, u = s["logits"], s["legal"], s["u"]
    B, A = logits.shape
    T, k, p, m = (_column(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    z = logits.double()
    ok = z > -math.inf                                   # false for NaN too
    if legal is not None:
        ok = ok & (legal != 0)
    z = torch.where(ok, z, -math.inf)
    top = z.amax(1, keepdim=True)
    some = ok.any(1, keepdim=True)
    d = torch.where(z == top, 0.0, z - top)              # <= 0
    greedy = torch.as_tensor(T == 0, device=z.device)
    x = torch.where(greedy, torch.where(d == 0, 0.0, -math.inf), d / T)
    w = torch.where(ok, torch.exp(x), 0.0)
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(A, device=z.device)[None, :]
    count = ok.sum(1, keepdim=True)
    k = torch.as_tensor(k, device=z.device)
    limit = torch.where(k > 0, torch.minimum(k.long(), count), count)
    limit = torch.where(greedy, torch.minimum(count, torch.ones_like(count)), limit)
    ins = rank < limit
    wk = torch.where(ins, ws, 0.0)
    cum = wk.cumsum(1)
    p = torch.as_tensor(p, dtype=torch.float64, device=z.device)
    keep = ins & ((p >= 1.0) | (cum - wk < p * cum[:, -1:])) & (ws >= m)
    kept = keep.sum(1).to(torch.int32)
    keep = torch.zeros_like(keep).scatter(1, order, keep)
    w = torch.where(keep, w, 0.0)
    c = w.cumsum(1)
    total = c[:, -1:]
    action = (c <= u[:, None] * total).sum(1, keepdim=True)
    last = torch.where(w > 0, rank, -1).amax(1, keepdim=True)
    action = torch.where(some, torch.minimum(action, last), -1)
    here = action.clamp(min=0)
    logprob = torch.where(some, x.gather(1, here) - torch.log(total), 0.0)
    r = dict(action=action[:, 0].to(torch.int32), logprob=logprob[:, 0].float(), kept=kept)
    if "probs" in s["out"]:
        r["probs"] = torch.where(some, w / total, 0.0).float()
    return r


def _plain_adapter(s):
    x, a, b, index = s["x"].float(), s["a"].float(), s["b"].float(), s["index"]
    n, r, K = a.shape
    y = x @ s["weight"].float().t()
    t = (x @ a.reshape(n * r, K).t()).reshape(-1, n, r)
    mine = (index[:, None] == torch.arange(n, device=x.device)[None, :]).float() * s["scale"][None, :]
    t = (t * mine[:, :, None]).reshape(-1, n * r)
    y = y + t @ b.permute(0, 2, 1).reshape(n * r, -1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def work(case):
    e = BYTES[case["dtype"]]
    B = case["rows"]
    if case["op"] == "sample":
        A = case["actions"]
        n = B * A * (e + (case["mask"] != "none") + (4 if case["probs"] else 0)) + B * (8 + 12)
        if case["per_row"]:
            n += B * (8 + (4 if case["top_k"] else 0) + (8 if case["top_p"] < 1 else 0) + (8 if case["min_p"] else 0))
        return dict(bytes=n, flops=4 * B * A)
    K, N, r, n = case["inner"], case["outer"], case["rank"], case["adapters"]
    used = min(n, B) if case["order"] == "distinct" else n * (1.0 - (1.0 - 1.0 / n) ** B)     # adapters that some row names
    used = used if case["bare"] == 0 else min(used, max(1.0, (1.0 - case["bare"]) * B))
    nbytes = e * (B * K + N * K + B * N + used * r * (K + N) + (N if case["bias"] else 0)) + 4 * (B + n)
    return dict(bytes=int(nbytes), flops=2 * B * K * N + int(2 * (1 - case["bare"]) * B * r * (K + N)))


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_sample(s) if s["op"] == "sample" else dict(y=_exact_adapter(s))


def _of_row(v, i):
    return v[i].item() if isinstance(v, torch.Tensor) else v


def _exact_sample(s):
    """Row by row on the host: rank the entries, cut the ranking at the shortest of the three prefixes, draw."""
    z_all = s["logits"].float().cpu().numpy().astype(np.float64)
    B, A = z_all.shape
    ok_all = ~np.isnan(z_all) & (z_all != -np.inf)
    if s["legal"] is not None:
        ok_all &= s["legal"].cpu().numpy() != 0
    u = s["u"].cpu().numpy()
    action, kept, logprob = np.full(B, -1, np.int32), np.zeros(B, np.int32), np.zeros(B, np.float64)
    probs = np.zeros((B, A), np.float64) if "probs" in s["out"] else None
    T, k, p, m = (s[n].cpu() if isinstance(s[n], torch.Tensor) else s[n] for n in ("temperature", "top_k", "top_p", "min_p"))
    for i in range(B):
        ids = np.flatnonzero(ok_all[i])
        if not len(ids):
            continue
        z = z_all[i, ids]
        ti, ki, pi, mi = (_of_row(v, i) for v in (T, k, p, m))
        if ti == 0:
            action[i], kept[i] = ids[np.argmax(z)], 1
            if probs is not None:
                probs[i, action[i]] = 1.0
            continue
        ranked = np.argsort(-z, kind="stable")
        x = (z[ranked] - z[ranked[0]]) / ti
        w = np.exp(x)
        n = min(ki, len(ids)) if ki > 0 else len(ids)
        if pi < 1:
            sums = np.cumsum(w[:n])
            n_p = 1 + int(np.searchsorted(sums, pi * sums[-1], side="left"))   # sums before an entry < p * all
            n = min(n, n_p)
        if mi > 0:
            n = min(n, int(np.sum(w >= mi)))
        chosen = np.sort(ranked[:n])
        weight = np.empty(len(ids))
        weight[ranked] = w
        c = np.cumsum(weight[chosen])
        j = int(np.searchsorted(c, u[i] * c[-1], side="right"))
        j = min(j, int(np.flatnonzero(weight[chosen])[-1]))
        action[i], kept[i] = ids[chosen[j]], n
        logprob[i] = (z[chosen[j]] - z[ranked[0]]) / ti - math.log(c[-1])
        if probs is not None:
            probs[i, ids[chosen]] = weight[chosen] / c[-1]
    r = dict(action=action, logprob=logprob, kept=kept)
    if probs is not None:
        r["probs"] = probs
    return r


def _exact_adapter(s):
    """Adapter by adapter, in 64 bits."""
    x, index = s["x"].double(), s["index"]
    y = torch.matmul(x, s["weight"].double().t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    for i in range(s["a"].shape[0]):
        rows = torch.nonzero(index == i)[:, 0]
        if len(rows):
            t = torch.matmul(x[rows], s["a"][i].double().t().contiguous())
            y[rows] += float(s["scale"][i]) * torch.matmul(t, s["b"][i].double().t().contiguous())
    return y

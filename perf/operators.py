"""Layer norm, cross attention and the relative position bias: the cases they are measured on, and their plain forms.

Kinds of a case ("kind"):
  layernorm  layer norm of rows; with "train" its backward pass too: y, and dx, dgamma, dbeta
  attention  attention of q [S][Lq][H][64] over k and v [S][Lk][KV heads][64] of another length; with "buckets" a
             learned relative position bias on the scores, with "train" the backward pass too: out, and dq, dk, dv
             and the bias table's gradient

Sizes: dim 384 with 8 heads and frames of 10 ms (801 in an 8 s window, 62 bands: 49662 tokens) are the benchmark
configuration's, dim 256 and 862 or 1723 frames the reference host's; the rest are generic.  Activations are N(0, 1),
gains N(1, 0.02), bias tables N(0, 1); scores have the factor 1/8, or q comes times 1/8 and the factor is 1.
"ragged": the sequences' key lengths fall evenly from the whole length to about a third of it, and from 8 sequences
on the last one is an empty slot (no key).
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
EPS = 1e-5
HEAD = 64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token's norm in a step of decoding: the latency of a call
        {"name": "norm_token", "kind": "layernorm", "type": "fp32", "rows": 1, "dim": 384, "train": False},
        # the tokens of an 8 s window, in the activations' reduced precision
        {"name": "norm_window_bf16", "kind": "layernorm", "type": "bf16", "rows": 49662, "dim": 384, "train": False},
        # a training step's norm of the same window
        {"name": "norm_train_fp32", "kind": "layernorm", "type": "fp32", "rows": 49662, "dim": 384, "train": True},
        # rows of an odd width, so that no two rows have the same alignment
        {"name": "norm_train_odd_bf16", "kind": "layernorm", "type": "bf16", "rows": 20011, "dim": 1023,
         "train": True},
        # one new token against a short text's states: the smallest call of a decoder's step
        {"name": "cross_step_fp32", "kind": "attention", "type": "fp32", "sequences": 1, "heads": 8, "kv_heads": 8,
         "q": 1, "k": 77, "ragged": False, "causal": False, "buckets": 0, "train": False},
        # single tokens of a batch of requests over long cached states, shared heads, one slot idle
        {"name": "cross_step_long_bf16", "kind": "attention", "type": "bf16", "sequences": 16, "heads": 32,
         "kv_heads": 8, "q": 1, "k": 8192, "ragged": True, "causal": False, "buckets": 0, "train": False},
        # the windows of a device pass against the reference track's frames, padded to the longest
        {"name": "cross_windows_bf16", "kind": "attention", "type": "bf16", "sequences": 8, "heads": 8,
         "kv_heads": 8, "q": 801, "k": 1723, "ragged": True, "causal": False, "buckets": 0, "train": False},
        # a training step of cross attention in full precision, odd lengths
        {"name": "cross_train_fp32", "kind": "attention", "type": "fp32", "sequences": 4, "heads": 8, "kv_heads": 8,
         "q": 801, "k": 389, "ragged": True, "causal": False, "buckets": 0, "train": True},
        # a training step of cross attention, shared heads
        {"name": "cross_train_bf16", "kind": "attention", "type": "bf16", "sequences": 8, "heads": 8, "kv_heads": 4,
         "q": 1023, "k": 862, "ragged": True, "causal": False, "buckets": 0, "train": True},
        # a decoder's step of its own attention: one token per sequence at the end of what it has written
        {"name": "bias_step_bf16", "kind": "attention", "type": "bf16", "sequences": 32, "heads": 12, "kv_heads": 12,
         "q": 1, "k": 512, "ragged": True, "causal": True, "buckets": 32, "max_distance": 128,
         "bidirectional": False, "train": False},
        # a training step of an encoder's own attention with the bias, and the table's gradient
        {"name": "bias_train_bf16", "kind": "attention", "type": "bf16", "sequences": 4, "heads": 12, "kv_heads": 12,
         "q": 1025, "k": 1025, "ragged": True, "causal": False, "buckets": 32, "max_distance": 128,
         "bidirectional": True, "train": True},
        # an encoder over long sequences: the largest
        {"name": "bias_long_bf16", "kind": "attention", "type": "bf16", "sequences": 4, "heads": 16, "kv_heads": 16,
         "q": 4096, "k": 4096, "ragged": False, "causal": False, "buckets": 32, "max_distance": 128,
         "bidirectional": True, "train": False},
    ]


def draw(rng):
    def between(lo, hi):  # log-uniform whole number
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["layernorm", "attention", "attention", "attention"])
    dtype = rng.choice(["fp32", "bf16"])
    train = rng.random() < 0.5
    if kind == "layernorm":
        dim = between(64, 8192)
        dim = rng.choice([dim, dim, max(64, dim // 64 * 64)])
        return {"kind": kind, "type": dtype, "rows": between(1, 20_000_000 // dim), "dim": dim, "train": train}
    step = not train and rng.random() < 0.4
    biased, causal = rng.random() < 0.5, rng.random() < 0.4
    kv_heads = rng.choice([1, 2, 4, 8, 8, 12, 16])
    heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
    case = {"kind": kind, "type": dtype, "sequences": between(1, 32), "heads": heads, "kv_heads": kv_heads,
            "q": rng.randint(1, 4) if step else between(16, 4096), "k": between(16, 8192 if step else 4096),
            "ragged": rng.random() < 0.6, "causal": causal, "buckets": 0, "train": train}
    if biased:
        case["bidirectional"] = not causal
        case["buckets"] = rng.choice([16, 32, 64])
        case["max_distance"] = rng.choice([96, 128, 256, 800])
    # at most the listed ones' scores (fp32 products run at a fraction of bf16's rate) and cache
    most = (3.0e8 if dtype == "bf16" else 6.0e7) * (0.15 if train else 1.0)
    while case["sequences"] * heads * case["q"] * case["k"] > most:
        if case["sequences"] > 1:
            case["sequences"] = (case["sequences"] + 1) // 2
        elif case["q"] > case["k"]:
            case["q"] = case["q"] * 2 // 3
        else:
            case["k"] = case["k"] * 2 // 3
    while case["sequences"] * kv_heads * case["k"] > (500_000 if dtype == "bf16" else 250_000):
        case["sequences"] = (case["sequences"] + 1) // 2
    return case


def _key_lengths(case):
    S, Lk = case["sequences"], case["k"]
    if not case["ragged"]:
        return [Lk] * S
    lengths = [max(1, Lk - (2 * Lk * s) // (3 * S)) for s in range(S)]
    if S >= 8:
        lengths[-1] = 0
    return lengths


def _is_step(case):
    return case["causal"] and not case["train"] and case["q"] <= 4


def _starts(case):
    """Position of each sequence's first query row among its keys: a step's new tokens are its last keys."""
    if not _is_step(case):
        return [0] * case["sequences"]
    return [max(0, n - case["q"]) for n in _key_lengths(case)]


# ---------------------------------------------------------------- inputs

def _randn(seed, stream, *shape):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 16 + stream) & 0x7FFFFFFFFFFF)
    return torch.randn(*shape, device=DEV, generator=g)


def _native():
    path = os.path.join(os.getcwd(), "karaoke-platform-sidecar-native_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vocalarc_hip import native
    return native


def _buffer(nbytes):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=DEV)


def prepare(case, seed):
    return _prepare_norm(case, seed) if case["kind"] == "layernorm" else _prepare_attention(case, seed)


def _prepare_norm(case, seed):
    rows, dim, t = case["rows"], case["dim"], TYPES[case["type"]]
    s = {"case": case, "x": (_randn(seed, 0, rows, dim) + 0.5).to(t),
         "gamma": 1 + 0.02 * _randn(seed, 1, dim), "beta": 0.02 * _randn(seed, 2, dim)}
    if case["train"]:
        s["dy"] = _randn(seed, 3, rows, dim).to(t)
    if own:  # what a program keeps: the context, outputs, row statistics and workspace
        native = _native()
        s["ctx"] = native.Context()
        s["y"] = torch.empty_like(s["x"])
        if case["train"]:
            s["stats"] = torch.empty(rows, 2, device=DEV)
            s["dx"], s["dgamma"], s["dbeta"] = torch.empty_like(s["x"]), torch.empty(dim, device=DEV), \
                torch.empty(dim, device=DEV)
            s["workspace"] = _buffer(native.Context.layernorm_workspace_bytes(rows, dim))
    return s


def _prepare_attention(case, seed):
    S, H, KV, Lq, Lk = (case[n] for n in ("sequences", "heads", "kv_heads", "q", "k"))
    t = TYPES[case["type"]]
    biased = case["buckets"] > 0
    q = _randn(seed, 0, S, Lq, H, HEAD)
    s = {"case": case, "q": (q / 8 if biased else q).to(t), "scale": 1.0 if biased else 0.125}
    if Lq <= 4:  # caches of keys and of values
        s["k"], s["v"] = _randn(seed, 1, S, Lk, KV, HEAD).to(t), _randn(seed, 2, S, Lk, KV, HEAD).to(t)
    else:  # one projection's k | v
        s["kv"] = _randn(seed, 1, S, Lk, 2, KV, HEAD).to(t)
        s["k"], s["v"] = s["kv"][:, :, 0], s["kv"][:, :, 1]
    if case["ragged"]:
        s["key_lengths"] = torch.tensor(_key_lengths(case), dtype=torch.int32, device=DEV)
    if _is_step(case):
        s["query_start"] = torch.tensor(_starts(case), dtype=torch.int32, device=DEV)
    if biased:
        s["table"] = _randn(seed, 3, case["buckets"], H)
    if case["train"]:
        s["dout"] = _randn(seed, 4, S, Lq, H, HEAD).to(t)
    if own:  # what a program keeps: the context, the attention's layout, outputs and workspaces
        native = _native()
        s["ctx"] = native.Context()
        s["out"] = torch.empty_like(s["q"])
        bias = {"bias_table": s["table"], "max_distance": case["max_distance"],
                "bidirectional": case["bidirectional"]} if biased else {}
        s["plan"] = p = native.CrossAttention(s["ctx"], s["q"], s["k"], s["v"], s["out"], causal=case["causal"],
                                              scale=s["scale"], key_lengths=s.get("key_lengths"),
                                              query_start=s.get("query_start"), **bias)
        s["workspace"] = _buffer(max(p.workspace_bytes(False), p.workspace_bytes(True) if case["train"] else 0))
        if case["train"]:
            s["saved"], s["dq"] = _buffer(p.saved_bytes()), torch.empty_like(s["q"])
            s["dkv"] = torch.empty_like(s["kv"]) if "kv" in s else None
            s["dk"] = s["dkv"][:, :, 0] if "kv" in s else torch.empty_like(s["k"])
            s["dv"] = s["dkv"][:, :, 1] if "kv" in s else torch.empty_like(s["v"])
            s["dtable"] = torch.empty_like(s["table"]) if biased else None
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    if s["case"]["kind"] == "layernorm":
        return _norm_own(s) if own else _norm_plain(s)
    return _attention_own(s) if own else _attention_plain(s)


def _norm_own(s):
    rows, dim, train = s["case"]["rows"], s["case"]["dim"], s["case"]["train"]
    bf16 = s["case"]["type"] == "bf16"
    s["ctx"].layernorm(s["x"], s["gamma"], s["beta"], s["y"], rows, dim, eps=EPS, stats=s.get("stats"), bf16=bf16)
    if not train:
        return {"y": s["y"]}
    s["ctx"].layernorm_backward(s["dy"], s["x"], s["gamma"], s["stats"], s["dx"], rows, dim, dgamma=s["dgamma"],
                                dbeta=s["dbeta"], workspace=s["workspace"], bf16=bf16)
    return {"y": s["y"], "dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}


def _norm_plain(s):
    t = s["x"].dtype
    x = s["x"].float()
    c = x - x.mean(-1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(-1, keepdim=True) + EPS)
    h = c * rstd
    y = (h * s["gamma"] + s["beta"]).to(t)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(t), "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0)}


def _attention_own(s):
    p, train = s["plan"], s["case"]["train"]
    p.forward(s["q"], s["k"], s["v"], s["out"], saved=s.get("saved"), workspace=s["workspace"])
    if not train:
        return {"out": s["out"]}
    p.backward(s["q"], s["k"], s["v"], s["out"], s["saved"], s["dout"], s["dq"], s["dk"], s["dv"], dbias=s["dtable"],
               workspace=s["workspace"])
    r = {"out": s["out"], "dq": s["dq"], "dk": s["dk"], "dv": s["dv"]}
    if s["dtable"] is not None:
        r["dtable"] = s["dtable"]
    return r


def _bucket(rel, case):
    """Bucket of each relative position (key's minus query's)."""
    side = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    near = side // 2
    n = rel.abs() if case["bidirectional"] else (-rel).clamp(min=0)
    # in 64 bits, and the borders' own distances (whole multiples of the logarithm's step) counted as reached
    steps = torch.log(n.clamp(min=near).double() / near) / math.log(case["max_distance"] / near) * (side - near)
    far = (near + torch.floor(steps + 1e-9).long()).clamp(max=side - 1)
    b = torch.where(n < near, n, far)
    return torch.where(rel > 0, b + side, b) if case["bidirectional"] else b


def _attention_plain(s):
    case, t = s["case"], s["q"].dtype
    H, KV, Lq, Lk = case["heads"], case["kv_heads"], case["q"], case["k"]
    q = s["q"].float().transpose(1, 2)  # [S][H][Lq][64]
    k = s["k"].float().repeat_interleave(H // KV, 2).transpose(1, 2)
    v = s["v"].float().repeat_interleave(H // KV, 2).transpose(1, 2)
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    at = torch.arange(Lk, device=DEV)
    pos = torch.arange(Lq, device=DEV)[None, :]
    if "query_start" in s:
        pos = pos + s["query_start"].long()[:, None]
    rel = at - pos[:, :, None]  # [S or 1][Lq][Lk]
    if case["buckets"]:
        x = x + s["table"][_bucket(rel, case)].permute(0, 3, 1, 2)
    visible = None
    if "key_lengths" in s:
        visible = (at < s["key_lengths"].long()[:, None])[:, None, None, :]
    if case["causal"]:
        past = (rel <= 0)[:, None]
        visible = past if visible is None else visible & past
    if visible is not None:
        x = x.masked_fill(~visible, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # finite where a row has no key
    p = torch.exp(x - m)
    p = p / p.sum(-1, keepdim=True).clamp(min=1.0)  # the largest adds 1: less only without a key
    out = torch.matmul(p, v).transpose(1, 2).to(t)
    if not case["train"]:
        return {"out": out}
    do = s["dout"].float().transpose(1, 2)
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dq = (torch.matmul(ds, k) * s["scale"]).transpose(1, 2).to(t)
    shared = lambda g: g.unflatten(1, (KV, H // KV)).sum(2).transpose(1, 2).to(t)  # noqa: E731
    r = {"out": out, "dq": dq, "dk": shared(torch.matmul(ds.transpose(2, 3), q) * s["scale"]),
         "dv": shared(torch.matmul(p.transpose(2, 3), do))}
    if case["buckets"]:
        # sums of the diagonals key - query = const: rows of Lq + Lk, read with a step of one less, put each
        # diagonal into a column; then the buckets' sums of those
        d = _columns(ds.sum(0))
        b = _bucket(torch.arange(d.shape[-1], device=DEV) - (Lq - 1), case)
        hot = (b[:, None] == torch.arange(case["buckets"], device=DEV)).double()
        r["dtable"] = torch.matmul(d.sum(1).double(), hot).t().float()
    return r


def _columns(x):
    """x [H][Lq][Lk] with x[h][i][j] in column j - i + Lq - 1 of Lq + Lk - 1."""
    H, Lq, Lk = x.shape
    wide = torch.nn.functional.pad(x.flip(1), (0, Lq)).flatten(1)  # rows Lq - 1 - i of Lk + Lq
    return wide[:, :Lq * (Lk + Lq - 1)].reshape(H, Lq, Lk + Lq - 1)


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["kind"] == "layernorm":
        n, dim = case["rows"] * case["dim"], case["dim"]
        if not case["train"]:
            return {"bytes": 2 * n * size + 8 * dim, "flops": 8 * n}
        return {"bytes": 4 * n * size + 16 * dim, "flops": 20 * n}
    S, H, KV, Lq, Lk = (case[n] for n in ("sequences", "heads", "kv_heads", "q", "k"))
    lengths, starts = _key_lengths(case), _starts(case)
    pairs = 0
    for n, start in zip(lengths, starts):
        if not case["causal"]:
            pairs += n * Lq
        else:  # row i sees min(n, start + i + 1)
            full = max(0, min(Lq, start + Lq - n + 1)) if n else 0  # rows that see all n
            first = Lq - full
            pairs += full * n + first * (start + 1) + first * (first - 1) // 2 if n else 0
    rows, keys = S * Lq * H * HEAD, sum(lengths) * KV * HEAD
    table = 4 * case["buckets"] * H
    if not case["train"]:
        return {"bytes": size * (2 * rows + 2 * keys) + table, "flops": 4 * HEAD * pairs * H}
    # q, k, v, dout read, out, dq, dk, dv written (dk, dv whole)
    return {"bytes": size * (4 * rows + 2 * keys + 2 * S * Lk * KV * HEAD) + 2 * table,
            "flops": 14 * HEAD * pairs * H}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _norm_exact(s) if case["kind"] == "layernorm" else _attention_exact(s)


def _norm_exact(s):
    x, gamma, beta = (s[n].double().requires_grad_() for n in ("x", "gamma", "beta"))
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = (x - mean) / (var + EPS).sqrt() * gamma + beta
    if not s["case"]["train"]:
        return {"y": y.detach()}
    dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _borders(case):
    """Distances at which the far buckets begin: n reaches step t when n^far >= max_distance^t near^(far - t)."""
    side = case["buckets"] // 2 if case["bidirectional"] else case["buckets"]
    near = side // 2
    far, top = side - near, case["max_distance"]
    found, n = list(range(1, near + 1)), near
    for t in range(1, far):
        while n ** far < top ** t * near ** (far - t):
            n += 1
        found.append(n)
    return torch.tensor(found, device=DEV)


def _attention_exact(s):
    case = s["case"]
    S, H, KV, Lq, Lk = (case[n] for n in ("sequences", "heads", "kv_heads", "q", "k"))
    train, lengths, starts = case["train"], _key_lengths(case), _starts(case)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    dq, dk, dv = torch.zeros_like(out), torch.zeros(s["k"].shape, dtype=torch.float64, device=DEV), \
        torch.zeros(s["v"].shape, dtype=torch.float64, device=DEV)
    dtable = torch.zeros(case["buckets"], H, dtype=torch.float64, device=DEV)
    for b in range(S):
        n = lengths[b]
        if not n:
            continue
        far = torch.arange(n, device=DEV) - torch.arange(starts[b], starts[b] + Lq, device=DEV)[:, None]
        bucket = None
        if case["buckets"]:
            if case["bidirectional"]:
                bucket = torch.bucketize(far.abs(), _borders(case), right=True) + (far > 0) * (case["buckets"] // 2)
            else:
                bucket = torch.bucketize((-far).clamp(min=0), _borders(case), right=True)
        for h in range(H):
            g = h // (H // KV)
            q, k, v = (a.double().requires_grad_() for a in (s["q"][b, :, h], s["k"][b, :n, g], s["v"][b, :n, g]))
            table = s["table"][:, h].double().requires_grad_() if bucket is not None else None
            x = (q @ k.t()) * s["scale"]
            if table is not None:
                x = x + table[bucket]
            if case["causal"]:
                x = torch.where(far > 0, -torch.inf, x)
            o = torch.softmax(x, -1) @ v  # every row of a sequence with keys sees one
            out[b, :, h] = o.detach()
            if not train:
                continue
            leaves = (q, k, v) + ((table,) if table is not None else ())
            grads = torch.autograd.grad(o, leaves, s["dout"][b, :, h].double())
            dq[b, :, h] = grads[0]
            dk[b, :n, g] += grads[1]
            dv[b, :n, g] += grads[2]
            if table is not None:
                dtable[:, h] += grads[3]
    if not train:
        return {"out": out}
    r = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if case["buckets"]:
        r["dtable"] = dtable
    return r

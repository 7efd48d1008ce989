"""Rotary positions, the paged cache, attention over it and beam search from their definitions, in 64 bits where a result is
rounded in its own way, and in 32 bits operation by operation where the library says how.  Roundings are counted as half
a step (U of fp32, HALF of a stored type) of what is rounded."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
BLOCK = 16


# ---------------------------------------------------------------- rotary positions

def theta(dim, base=10000.0, factor=1.0, original=0, low=1.0, high=32.0):
    t = [base ** (-2 * i / dim) for i in range(dim // 2)]
    if factor > 1:
        keep = [min(1.0, max(0.0, (original * x / (2 * math.pi) - low) / (high - low))) if original else 0.0 for x in t]
        t = [x * (k + (1 - k) / factor) for x, k in zip(t, keep)]
    return torch.tensor(t, dtype=torch.float64)


def pairs(x, dim, interleaved):
    """The two halves [..., dim / 2] of the pairs, and the rest."""
    r, rest = x[..., :dim], x[..., dim:]
    return (r[..., 0::2], r[..., 1::2], rest) if interleaved else (r[..., :dim // 2], r[..., dim // 2:], rest)


def unpairs(a, b, rest, interleaved):
    r = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((r, rest), -1)


def rotary(x, start, dim, interleaved, backward=False, magnitude=1.0, **angles):
    """x [S][L][H][D] on the CPU -> (value, bound) in 64 bits."""
    S, L = x.shape[:2]
    p = torch.tensor(start, dtype=torch.float64)[:, None] + torch.arange(L)
    angle = (p[..., None] * theta(dim, **angles))[:, :, None]
    c, s = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if backward else 1)
    a, b, rest = pairs(x.double(), dim, interleaved)
    u, w = a * c - b * s, a * s + b * c
    # the table's entries, the products and the sum are rounded once each; angles in 64 bits are off by 2^-52 of them
    loose = 2.02 * U + 2.0 ** -50 * (1 + p.abs().max().item())
    du, dw = loose * ((a * c).abs() + (b * s).abs()) + U * u.abs(), loose * ((a * s).abs() + (b * c).abs()) + U * w.abs()
    wide = 2.0 ** -50 * (1 + p.abs().max().item()) * (a.abs() + b.abs())  # near a zero of the cosine
    val = unpairs(u, w, rest, interleaved)
    tol = unpairs(du + wide, dw + wide, torch.zeros_like(rest), interleaved)
    if x.dtype == torch.bfloat16:
        tol = tol * 1.01 + HALF[x.dtype] * val.abs()
        tol[..., dim:] = 0
    return val, tol


def turn32(x, table, start, interleaved):
    """x [L][H][D] fp32 turned by the table's own rows from position start on, each product and sum rounded."""
    dim = 2 * table.shape[1]
    cs = table[start:start + x.shape[0]][:, None]
    a, b, rest = pairs(x, dim, interleaved)
    return unpairs(a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0], rest, interleaved)


# ---------------------------------------------------------------- the cache

class Cache:
    """What each sequence's cache holds, in 32 bits as the library says: numbers and scales, or bf16 values."""

    def __init__(self, kind, sequences, kv_heads, head_dim):
        self.kind, self.n = kind, [0] * sequences
        # per sequence and part, tokens by heads: numbers (or values), and per block of tokens the scale of each head
        self.q = [[torch.zeros(0, kv_heads, head_dim) for _ in "kv"] for _ in range(sequences)]
        self.s = [[torch.zeros(0, kv_heads) for _ in "kv"] for _ in range(sequences)]

    def append(self, s, start, k, v):
        """k (already turned) and v [n][H][D] fp32 from position `start` on."""
        n = k.shape[0]
        if n == 0:
            return
        end = -(-(start + n) // BLOCK) * BLOCK
        for part, x in enumerate((k, v)):
            q, sc = self.q[s][part], self.s[s][part]
            if q.shape[0] < end:
                q = torch.cat((q, torch.zeros(end - q.shape[0], *q.shape[1:])))
                sc = torch.cat((sc, torch.zeros(end // BLOCK - sc.shape[0], sc.shape[1])))
            for b in range(start // BLOCK, end // BLOCK):
                lo, hi = max(start - b * BLOCK, 0), min(start + n - b * BLOCK, BLOCK)
                new = x[b * BLOCK + lo - start:b * BLOCK + hi - start]
                rows = q[b * BLOCK:(b + 1) * BLOCK]
                rows[hi:] = 0
                if self.kind == "bf16":
                    rows[lo:hi] = new.bfloat16().float()
                    continue
                scale = (new.abs().amax((0, 2)) * torch.tensor(1 / 127)).clamp(min=2.0 ** -100)
                if lo:
                    scale = torch.maximum(scale, sc[b])
                inv = 1 / scale
                if lo:
                    rows[:lo] = torch.round(rows[:lo] * (sc[b] * inv)[:, None])
                rows[lo:hi] = torch.round(new * inv[:, None]).clamp(-127, 127)
                sc[b] = scale
            self.q[s][part], self.s[s][part] = q, sc
        self.n[s] = start + n

    def values(self, s, part, upto=None):
        q = self.q[s][part]
        if self.kind == "int8":
            q = q * self.s[s][part].repeat_interleave(BLOCK, 0)[..., None]
        return q[:self.n[s] if upto is None else upto]


# ---------------------------------------------------------------- attention

def attention(kind, q, keys, values, *, scale, causal=False, start=0, turn=None, operand=None):
    """q [L][H][D] of one sequence over keys and values [n][KV][D] (any type, 64 bits inside) -> (value, bound).
    turn: the queries' rotation in 64 bits, q -> q'.  kind: of the cache; the queries' type says how it is rounded.  operand:
    what a value of q' and of P may be off by as an operand, where a test holds it to less."""
    dtype = q.dtype
    L, H, D = q.shape
    n, KV = keys.shape[:2]
    val, tol = torch.zeros(L, H, D, dtype=torch.float64), torch.zeros(L, H, D, dtype=torch.float64)
    q64 = turn(q) if turn else q.double()
    # what a value of q' and of P is off by as an operand: fp16 2^-11 a piece, bf16 2^-8
    piece, pieces = (2.0 ** -11, 1 if dtype == torch.bfloat16 else 2) if kind == "int8" else \
        (2.0 ** -8, 1 if dtype == torch.bfloat16 else 3)
    operand = max(piece ** pieces, U) if operand is None else operand
    for h in range(H):
        g = h // (H // KV)
        qh, k, v = q64[:, h], keys[:, g].double(), values[:, g].double()
        x = qh @ k.t() * scale
        seen = torch.ones(L, n, dtype=torch.bool)
        if causal:
            seen = torch.arange(n) <= start + torch.arange(L)[:, None]
        empty = ~seen.any(1)
        x = x.masked_fill(~seen, -math.inf)
        p = torch.softmax(x.masked_fill(empty[:, None], 0), 1) * (~empty[:, None])
        out = p @ v
        # scores: q' as turned (4 roundings) and as an operand, fp16's smallest a 2^-38 of the row's largest, D / 32 + 8
        # additions, the scales' products
        size = qh.abs() @ k.abs().t() * abs(scale)
        tiny = qh.abs().amax(1, keepdim=True) * 2.0 ** -38 * k.abs().sum(1) * abs(scale) if kind == "int8" else 0
        dx = size * (operand + U * (D / 32 + 16)) + tiny + x.masked_fill(~seen, 0).abs() * 6 * U
        dx = dx.masked_fill(~seen, 0)
        # a probability: its score's error, its exponential's, its place as an operand; the sum's is at most that
        top = dx.amax(1, keepdim=True) if n else torch.zeros(L, 1, dtype=torch.float64)
        rel = 2 * torch.expm1(top) + operand + U * (n / 32 + 60)
        # P (times its block's scale over the largest) is fp16 times 2^10: below fp16's normal numbers it is off by up to half
        # of their step 2^-24, 2^-35 of the largest value, and the second operand's by as much
        small = n * 2.0 ** -34 * v.abs().amax() if kind == "int8" and n else 0
        val[:, h] = out
        tol[:, h] = rel * (p @ v.abs()) + small + HALF[dtype] * out.abs() * 1.01
    return val, tol


# ---------------------------------------------------------------- beam search

def beams(logits, scores, picks, end_token=-1, ended=None):
    """One sequence: logits [B][V], scores [B] -> picks of (score, beam, token) in the order that the header gives, and the
    smallest distance of two different scores among the first picks + 1."""
    B, V = logits.shape
    found = []
    for b in range(B):
        x, s = logits[b].double(), float(scores[b])
        lse = float(torch.logsumexp(x, 0))
        if ended is not None and ended[b] and math.isfinite(s):
            row = [(s if t == end_token else -math.inf, 0.0, t) for t in range(V)]
        elif not math.isfinite(s) or not math.isfinite(lse) or (ended is not None and ended[b]):
            row = [(-math.inf, 0.0, t) for t in range(V)]
        else:
            row = [(s + (float(v) - lse), float(v) if math.isfinite(float(v)) else 0.0, t) for t, v in enumerate(x)]
        row.sort(key=lambda c: (-c[0], -c[1], c[2]))
        found += [(c[0], b, c[1], c[2]) for c in row[:picks + 1]]
    found.sort(key=lambda c: (-c[0], c[1], -c[2], c[3]))
    near = [a[0] - b[0] for a, b in zip(found[:picks], found[1:picks + 1]) if a[1] != b[1] and math.isfinite(a[0])]
    return [(c[0], c[1], c[3]) for c in found[:picks]], min(near, default=math.inf)


def assert_within(got, val, tol, what):
    got = got.double().cpu()
    assert got.shape == val.shape, (what, got.shape, val.shape)
    off = (got - val).abs()
    bad = ~(off <= tol)
    if bad.any():
        i = (off / tol.clamp(min=1e-300)).nan_to_num(nan=math.inf).flatten().argmax()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond their bounds; worst {got.flatten()[i]} for "
                             f"{val.flatten()[i]}, bound {tol.flatten()[i]}")

"""Layer norm and attention with a relative position bias in 64 bits, from their definitions, each result with how far
the kernels' may be from it: every rounding counted as half a step (U of fp32, HALF of bf16) of what is rounded."""

from __future__ import annotations

import math

import torch

U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8}  # of a stored or multiplied value beyond fp32's own


def layernorm(x, gamma, beta, eps, dy=None):
    """({name: value}, {name: bound}); depth: additions that one sum passes through."""
    half = HALF[x.dtype] + U
    x64, g64 = x.double(), gamma.double()
    rows, dim = x.shape
    depth = dim / 64 + 16
    mu = x64.mean(-1, keepdim=True)
    c = x64 - mu
    rstd = 1 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    h = c * rstd
    b64 = beta.double() if beta is not None else torch.zeros_like(g64)
    y = h * g64 + b64
    # the mean is off by depth roundings of |x|, rstd by half as many of itself
    dh = U * (depth * rstd * x64.abs().mean(-1, keepdim=True) + (depth / 2 + 6) * h.abs())
    val, tol = {"y": y}, {"y": dh * g64.abs() * 1.01 + 2 * U * (y.abs() + b64.abs()) + half * y.abs()}
    if dy is None:
        return val, tol
    dy64 = dy.double()
    g = dy64 * g64
    c1, c2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = rstd * (g - c1 - h * c2)
    m = lambda t: t.abs().mean(-1, keepdim=True)  # noqa: E731
    ddx = rstd * (U * (depth + 8) * (g.abs() + m(g) + h.abs() * m(g * h)) + dh * c2.abs() + h.abs() * m(g * dh))
    # a workgroup's rows one after the other, then its part among 512
    adds = rows / 512 + 140
    val.update(dx=dx, dgamma=(dy64 * h).sum(0), dbeta=dy64.sum(0))
    tol.update(dx=1.01 * ddx + half * dx.abs(), dgamma=U * adds * (dy64 * h).abs().sum(0) + (dy64.abs() * dh).sum(0),
               dbeta=U * adds * dy64.abs().sum(0))
    return val, tol


def borders(buckets, max_distance, bidirectional):
    """Distances from which a side's buckets 1, 2, ... begin, in whole numbers: near buckets hold one distance each, and
    far bucket near + t begins at the first n with n^far >= max_distance^t near^(far - t)."""
    side = buckets // 2 if bidirectional else buckets
    near = side // 2
    far = side - near
    found, n = list(range(1, near + 1)), near
    for t in range(1, far):
        while n ** far < max_distance ** t * near ** (far - t):
            n += 1
        found.append(n)
    return found


def bucket(rel, buckets, max_distance, bidirectional):
    n = rel.abs() if bidirectional else (-rel).clamp(min=0)
    b = torch.bucketize(n, torch.tensor(borders(buckets, max_distance, bidirectional), device=rel.device), right=True)
    return b + (rel > 0) * (buckets // 2) if bidirectional else b


def attention(q, k, v, *, causal=False, scale=0.125, query_lengths=None, key_lengths=None, query_start=None,
              bias_table=None, max_distance=128, bidirectional=True, dout=None):
    """({name: value}, {name: bound}) of out, and with dout of dq, dk, dv and dbias."""
    S, Lq, H, D = q.shape
    Lk, KV = k.shape[1:3]
    half = HALF[q.dtype]
    lens = lambda t, most: [most] * S if t is None else [min(max(int(n), 0), most) for n in t]  # noqa: E731
    qlens, klens = lens(query_lengths, Lq), lens(key_lengths, Lk)
    starts = [0] * S if query_start is None else [int(n) for n in query_start]
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    val = {"out": zero(q)}
    if dout is not None:
        val.update(dq=zero(q), dk=zero(k), dv=zero(v))
        if bias_table is not None:
            val["dbias"] = zero(bias_table)
    tol = {n: torch.zeros_like(t) for n, t in val.items()}
    for s in range(S):
        m, n = qlens[s], klens[s]
        if not m or not n:
            continue
        i = torch.arange(m, device=q.device)[:, None] + starts[s]
        rel = torch.arange(n, device=q.device)[None, :] - i
        which = bucket(rel, bias_table.shape[0], max_distance, bidirectional) if bias_table is not None else None
        for h in range(H):
            g = h // (H // KV)
            Q, K, V = q[s, :m, h].double(), k[s, :n, g].double(), v[s, :n, g].double()
            x = Q @ K.t() * scale
            dx = 68 * U * abs(scale) * (Q.abs() @ K.abs().t())  # of a score: 64 products and sums, scale
            if which is not None:
                b = bias_table[:, h].double()[which]
                x = x + b
                dx = dx + 2 * U * torch.where(torch.isfinite(x), x.abs(), 0.0).clamp(max=1e6)
            if causal:
                x = x.masked_fill(rel > 0, -math.inf)
            top = x.amax(-1, keepdim=True)
            e = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
            l = e.sum(-1, keepdim=True)
            P = torch.where(l > 0, e / l, 0.0)
            O = P @ V
            # of a probability, of itself: its score, the row's (its sum), the exponentials' arguments and roundings
            gap = (torch.where(torch.isfinite(x), (top - x), 0.0)).clamp(0, 100)
            # and below 2^-126, fp32's smallest normal number, 0 may stand for it: exp(x - m) <= 1 and their sum >= 1,
            # so a probability is off by at most as much (a score 88 below its row's maximum)
            rp = dx + dx.amax(-1, keepdim=True) + U * (4 * gap + n / 8 + 24)
            dPr = P * rp + 2.0 ** -126
            PV = P @ V.abs()
            acc = dPr @ V.abs() + U * (n / 8 + 16) * PV  # of out's fp32 sums
            val["out"][s, :m, h] = O
            tol["out"][s, :m, h] = acc + half * PV + (half + U) * O.abs()
            if dout is None:
                continue
            dO = dout[s, :m, h].double()
            dP = dO @ V.t()
            delta = (dO * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            ddelta = (dO.abs() * (acc + 2 * half * half * (PV + O.abs()))).sum(-1, keepdim=True) + \
                70 * U * (dO * O).abs().sum(-1, keepdim=True)
            ddS = dPr * (dP - delta).abs() + P * (68 * U * (dO.abs() @ V.abs().t()) + ddelta) + 3 * U * dS.abs()
            sums = U * (max(m, n) / 8 + 16) + half  # of a product over rows or keys, and its operand's rounding
            val["dq"][s, :m, h] = dS @ K * scale
            tol["dq"][s, :m, h] = abs(scale) * ((ddS + sums * dS.abs()) @ K.abs())
            val["dk"][s, :n, g] += dS.t() @ Q * scale
            tol["dk"][s, :n, g] += abs(scale) * ((ddS + sums * dS.abs()).t() @ Q.abs())
            val["dv"][s, :n, g] += P.t() @ dO
            tol["dv"][s, :n, g] += (dPr + sums * P).t() @ dO.abs()
            if which is not None:
                # a tile's diagonal, the tiles' diagonals, 128 slots, the workgroups
                adds = U * (40 + n / 16 + 128 + S * (m / 128 + 1))
                for b in range(bias_table.shape[0]):
                    at = which == b
                    val["dbias"][b, h] += (dS * at).sum()
                    tol["dbias"][b, h] += ((ddS + adds * dS.abs()) * at).sum()
    for name in ("dq", "dk", "dv"):
        if name in val:
            tol[name] += (half + U) * (val[name].abs() + tol[name])
    return val, tol


def assert_within(got, val, tol, what=""):
    """Every element within its bound (and, past the bounds of fp32's range, as the value)."""
    g = got.double()
    assert g.shape == val.shape, f"{what}: shape {tuple(g.shape)}, not {tuple(val.shape)}"
    off = (g - val).abs()
    bad = ~(off <= tol + 1e-37)
    if bool(bad.any()):
        i = int(torch.where(bad, off / (tol + 1e-37), 0.0).nan_to_num(math.inf).flatten().argmax())
        at = tuple(int(a) for a in torch.unravel_index(torch.tensor(i), g.shape))
        raise AssertionError(f"{what}: {int(bad.sum())} of {g.numel()} out of bounds; worst at {at}: {g[at].item()!r}, "
                             f"not {val[at].item()!r} within {tol[at].item():.3g}")

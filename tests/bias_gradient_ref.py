"""Gradients of attention with a relative position bias in 64 bits, and how far off in norm a kernel's may be when every
rounding is independent of the others and evenly spread within its half step.

norm_cross_ref's bounds add up each pair's worst case, which over a bucket of millions of pairs is thousands of times what
such errors add up to.  Here their squares are added.  A value v, as often at one place of its binade as at another by
its logarithm, is rounded by up to U |v| / m, m in 1 .. 2: the mean of 1 / m^2 is 3 / (8 ln 2), and a third of the square is
the variance.  The limit is twice the resulting standard deviation: a norm of hundreds of such sums is within some
percent of it."""

from __future__ import annotations

import math

import torch

import norm_cross_ref as R

U = R.U
LN2 = math.log(2.0)


def pairs(q, k, v, table, dout, bucket, scale, causal, rel):
    """One (sequence, head) in 64 bits: (P, dS, delta, scores in powers of two with their parts)."""
    s = q @ k.t()
    x = s * scale + table[bucket]
    if causal:
        x = x.masked_fill(rel > 0, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isfinite(top), top, 0.0))
    l = e.sum(-1, keepdim=True)
    P = torch.where(l > 0, e / l, 0.0)
    dP = dout @ v.t()
    delta = (P * dP).sum(-1, keepdim=True)
    return s, x, top, l, P, dP, delta, P * (dP - delta)


def gradients(q, k, v, dout, *, bias_table, max_distance=128, bidirectional=True, causal=False, scale=0.125,
              key_lengths=None, query_start=None):
    """({name: value}, {name: limit of the norm of the difference}) of dq, dk, dv and dbias."""
    S, Lq, H, _ = q.shape
    Lk, KV = k.shape[1:3]
    half = R.HALF[q.dtype]
    adds = 64 if half else 6 * 64  # of a product over a head: fp32 in six products of pieces
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    val = {"dq": zero(q), "dk": zero(k), "dv": zero(v), "dbias": zero(bias_table)}
    var = {n: 0.0 for n in val}
    for s in range(S):
        n = Lk if key_lengths is None else int(key_lengths[s])
        if not n:
            continue
        at = torch.arange(n, device=q.device)[None, :]
        rel = at - torch.arange(Lq, device=q.device)[:, None] - (0 if query_start is None else int(query_start[s]))
        which = R.bucket(rel, bias_table.shape[0], max_distance, bidirectional)
        near = rel.abs() < max_distance + 64  # in tiles that are not wholly beyond max_distance, and a tile's width
        for h in range(H):
            g = h // (H // KV)
            Q, K, V, dO = (t.double() for t in (q[s, :, h], k[s, :n, g], v[s, :n, g], dout[s, :, h]))
            table = bias_table[:, h].double()
            sc, x, top, l, P, dP, delta, dS = pairs(Q, K, V, table, dO, which, scale, causal, rel)
            val["dq"][s, :, h] = dS @ K * scale
            val["dk"][s, :n, g] += dS.t() @ Q * scale
            val["dv"][s, :n, g] += P.t() @ dO
            val["dbias"][:, h].index_add_(0, which.flatten(), dS.flatten())
            seen = torch.isfinite(x)
            x2, m2, n2 = torch.where(seen, x, 0.0) / LN2, torch.where(torch.isfinite(top), top, 0.0) / LN2, l.log2()
            low = torch.where(seen, x2 - m2, 0.0)
            # squares of the largest half steps, in units of U.  Of a probability, of itself: the score's sum of 64 products (partial
            # sums of half its spread on average), factor and bias, the argument's two sums, exp2 (a whole step), and the
            # row's own sum of up to n / 2 + 16 terms in a lane, rising evenly
            spread = (Q * Q) @ (K * K).t()
            p2 = LN2 ** 2 * ((scale / LN2) ** 2 * adds / 2 * spread + (sc * scale / LN2) ** 2 + (table[which] / LN2) ** 2 +
                             x2 ** 2 + low ** 2 + (low - n2) ** 2) + 4 + (n / 2 + 16) / 3
            # of dP - delta, which one sum makes
            d2 = adds / 2 * ((dO * dO) @ (V * V).t()) + adds * delta ** 2
            e2 = torch.where(seen, P * P * d2 + dS * dS * (p2 + 1), 0.0)
            # of delta, the same in all of a row's pairs: out's sums over the keys (three products with P, fp32 six), their
            # product with dout, and the probabilities that the forward had
            o2 = (3 if half else 6) * n / 2 * ((P @ V) ** 2 + (P * P) @ (V * V))
            row2 = (dO * dO * (o2 + 32 * (P @ V) ** 2)).sum(-1, keepdim=True) + (P * P * dP * dP * p2).sum(-1, keepdim=True)
            # and what the operands' rounding takes where dS and P enter products, and the products' own sums
            cut = (half / U) ** 2
            sums = lambda n: cut + (3 if half else 6) * n / 2 + 16  # noqa: E731
            var["dq"] += float((scale ** 2 * ((e2 + sums(n) * dS * dS) @ (K * K) + row2 * (P @ K) ** 2)).sum())
            var["dk"] += float((scale ** 2 * ((e2 + sums(Lq) * dS * dS + P * P * row2).t() @ (Q * Q))).sum())
            var["dv"] += float(((P * P * (p2 + sums(Lq))).t() @ (dO * dO)).sum())
            # the table's: a lane's sum of 16 a tile over its tiles, then 60 more to join lanes, waves and workgroups; a
            # row's residual, which all its pairs' errors are in, comes out of the far buckets, so that these have it too;
            # delta's stays in the near ones
            var["dbias"] += float((2 * e2 + (n / 32 + 76) / 2 * dS * dS).sum() +
                                  (row2 * (P * near).sum(-1, keepdim=True) ** 2).sum())
    for name in ("dq", "dk", "dv"):
        var[name] += (half / U + 1) ** 2 * float(val[name].square().sum())
    return val, {n: 2 * U * math.sqrt(3 / (8 * LN2) / 3 * t) for n, t in var.items()}


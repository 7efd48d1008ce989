"""bias_gradient_ref's limits have teeth: fp32 arithmetic passes them, mistakes do not."""

import math

import pytest
import torch

import bias_gradient_ref as B
import norm_cross_ref as R

SIZE = (1, 2, 1, 300, 1100)


def table_gradient(q, k, v, dout, table, mistake):
    """By the kernels' formulas in fp32, with what the forward pass would keep of out."""
    _, Lq, H, _ = q.shape
    Lk, KV = k.shape[1:3]
    rel = torch.arange(Lk)[None, :] - torch.arange(Lq)[:, None]
    which = R.bucket(rel, 32, 128, True)
    g = torch.zeros(32, H, dtype=torch.float64)
    for h in range(H):
        Q, K, V, dO = (t.float() for t in (q[0, :, h], k[0, :, h * KV // H], v[0, :, h * KV // H], dout[0, :, h]))
        x = Q @ K.t() * 0.125 + table[:, h][which]
        m = x.amax(-1, keepdim=True)
        e = torch.exp(x - m)
        l = e.sum(-1, keepdim=True)
        out = (e.bfloat16().float() if mistake == "rounded P in out" else e) @ V / l
        if mistake == "rounded out":
            out = out.bfloat16().float()
        P = torch.exp((x - m) - torch.log(l))
        dP = dO @ V.t()
        dS = P * (dP - (dO * out).sum(-1, keepdim=True))
        if mistake == "rounded dS":
            dS = dS.bfloat16().float()
        dS = dS.double()
        far = torch.where(rel.abs() >= 128, P.double(), 0.0) * dS.sum(-1, keepdim=True)
        if mistake == "one bucket off":
            dS = dS.roll(1, 1)
        g[:, h].index_add_(0, which.flatten(), (dS - far).flatten())
    return g


@pytest.mark.parametrize("mistake", ["", "rounded out", "rounded P in out", "rounded dS", "one bucket off"])
def test_limits(mistake):
    S, H, KV, Lq, Lk = SIZE
    g = torch.Generator().manual_seed(3)
    r = lambda *shape: torch.randn(*shape, generator=g)  # noqa: E731
    q, k, v, dout = (t.bfloat16() for t in (r(S, Lq, H, 64), r(S, Lk, KV, 64), r(S, Lk, KV, 64), r(S, Lq, H, 64)))
    table = r(32, H)
    val, limit = B.gradients(q, k, v, dout, bias_table=table)
    off = float((table_gradient(q, k, v, dout, table, mistake) - val["dbias"]).norm())
    assert (off <= limit["dbias"]) == (not mistake), (off, limit["dbias"])


@pytest.mark.parametrize("causal", [False, True])
def test_values(causal):
    """The values are norm_cross_ref's, and their limits far below its bounds'."""
    g = torch.Generator().manual_seed(4)
    q, k, v, dout = (torch.randn(2, n, h, 64, generator=g) for n, h in ((70, 4), (300, 2), (300, 2), (70, 4)))
    kw = dict(bias_table=torch.randn(32, 4, generator=g), causal=causal, bidirectional=not causal, key_lengths=[300, 211],
              query_start=[230, 100] if causal else None)
    val, tol = R.attention(q, k, v, dout=dout, **kw)
    mine, limit = B.gradients(q, k, v, dout, **kw)
    for n in mine:
        assert torch.allclose(mine[n], val[n], rtol=1e-10, atol=1e-10), n
        assert 0 < limit[n] < (0.01 if n == "dbias" else 0.2) * float(tol[n].norm()), n
        assert math.isfinite(limit[n])

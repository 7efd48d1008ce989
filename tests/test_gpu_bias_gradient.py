"""The bias table's gradient where most of a row's keys are in the far buckets: against 64 bits in norm
(bias_gradient_ref.py), and how an error that all pairs of a row have in common spreads, in every cut of the work."""

import math

import pytest
import torch

import bias_gradient_ref as B
import norm_cross_ref as R
from helpers import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    from vocalarc_hip import native

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ctx():
    c = native.Context()
    yield c
    c.close()


def make(S, H, KV, Lq, Lk, dtype, buckets=32):
    g = torch.Generator(device=DEV)
    g.manual_seed(S * 1000 + Lq)
    r = lambda *shape: torch.randn(*shape, device=DEV, generator=g)  # noqa: E731
    return (r(S, Lq, H, 64).to(dtype), r(S, Lk, KV, 64).to(dtype), r(S, Lk, KV, 64).to(dtype), r(S, Lq, H, 64).to(dtype),
            r(buckets, H))


def buffer(n):
    return torch.empty(n, dtype=torch.uint8, device=DEV).fill_(0xff)


class Step:
    """Forward once, then the gradients from any out."""

    def __init__(self, ctx, q, k, v, dout, **kw):
        for n in ("key_lengths", "query_start"):
            if kw.get(n) is not None:
                kw[n] = torch.tensor(kw[n], dtype=torch.int32, device=DEV)
        self.t, self.dout, self.table, self.out = (q, k, v), dout, kw["bias_table"], torch.empty_like(q)
        self.p = native.CrossAttention(ctx, q, k, v, self.out, **kw)
        self.saved, self.ws = buffer(self.p.saved_bytes()), buffer(self.p.workspace_bytes(True))
        self.p.forward(q, k, v, self.out, saved=self.saved, workspace=buffer(self.p.workspace_bytes()))

    def gradients(self, out=None):
        r = dict(zip(("dq", "dk", "dv", "dbias"), (torch.full_like(t, math.nan) for t in self.t + (self.table,))))
        self.p.backward(*self.t, self.out if out is None else out, self.saved, self.dout, r["dq"], r["dk"], r["dv"],
                        dbias=r["dbias"], workspace=self.ws)
        return r


# (sequences, heads, key heads, rows, keys): workgroups of 128 rows, of 32, the same with the keys in 9 or in 2 pieces,
# single tokens in many pieces, short keys under many rows
SIZES = [(4, 12, 12, 1025, 1025), (2, 4, 2, 1025, 1025), (1, 8, 8, 200, 4096), (2, 8, 4, 500, 1500), (2, 4, 4, 1, 6000),
         (14, 8, 8, 4089, 60)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_norm(ctx, size, causal, dtype):
    S, _, _, Lq, Lk = size
    q, k, v, dout, table = make(*size, dtype)
    kw = dict(bias_table=table, bidirectional=not causal, causal=causal,
              key_lengths=[max(1, Lk - Lk * s // (2 * S)) for s in range(S)],
              query_start=[max(0, Lk - Lq - 5 * s) for s in range(S)] if causal else None)
    got = Step(ctx, q, k, v, dout, **kw).gradients()
    val, limit = B.gradients(q, k, v, dout, **kw)
    off = {n: float((got[n].double() - val[n]).norm()) for n in val}
    print(size, dtype, {n: "%.2e of %.2e" % (off[n] / float(val[n].norm()), limit[n] / float(val[n].norm())) for n in val})
    assert all(off[n] <= limit[n] for n in val), (off, limit)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size", [(4, 12, 12, 600, 1025), (2, 4, 2, 1025, 1025), (1, 8, 8, 200, 4096), (2, 8, 4, 500, 1500),
                                  (1, 1, 1, 33, 3000), (2, 4, 4, 1, 6000), (3, 2, 2, 70, 2000)], ids=str)
def test_rows_error_stays_out_of_the_far_buckets(ctx, size, causal, dtype):
    """out moved so that dout.out grows by e in every row: dS = P (dP - dout.out) is off by -e P, what a row's dS add up
    to by -e, and a side's last bucket has it taken out again but for the tiles that reach less than 64 past max_distance.
    Without that it would be off by e times all of its probability, more than 3 times as much on one side at least."""
    S, H, KV, Lq, Lk = size
    q, k, v, dout, table = make(*size, dtype)
    starts = [Lk - Lq - 5 * s for s in range(S)] if causal else [0] * S
    lens = [Lk - 40 * s for s in range(S)]
    kw = dict(bias_table=table, bidirectional=not causal, causal=causal, key_lengths=lens,
              query_start=starts if causal else None)
    step = Step(ctx, q, k, v, dout, **kw)
    d64 = dout.double()
    moved = (step.out.double() + d64 / d64.square().sum(-1, keepdim=True)).to(dtype)
    e = ((moved.double() - step.out.double()) * d64).sum(-1)  # [S][Lq][H], 1 but for bf16's roundings
    change = step.gradients(moved)["dbias"].double() - step.gradients()["dbias"].double()
    last = (31,) if causal else (15, 31)  # of a side
    whole, part = torch.zeros(2, H, dtype=torch.float64, device=DEV), torch.zeros(2, H, dtype=torch.float64, device=DEV)
    for s in range(S):
        rel = torch.arange(lens[s], device=DEV)[None, :] - torch.arange(Lq, device=DEV)[:, None] - starts[s]
        which = R.bucket(rel, 32, 128, not causal)
        for h in range(H):
            P = B.pairs(*(t.double() for t in (q[s, :, h], k[s, :lens[s], h * KV // H], v[s, :lens[s], h * KV // H])),
                        table[:, h].double(), d64[s, :, h], which, 0.125, causal, rel)[4]
            pe = P * e[s, :, h, None].abs()
            for i, b in enumerate(last):
                whole[i, h] += (pe * (which == b)).sum()
                part[i, h] += (pe * ((which == b) & (rel.abs() < 192))).sum()
    assert bool((whole.sum(1) > 3 * part.sum(1)).any())
    for i, b in enumerate(last):
        # fp32's roundings of what is taken out: sums of up to 2^13 additions in a chain, each half a step
        bound = 1.01 * part[i] + 2 ** 13 * R.U * whole[i]
        assert bool((change[b].abs() <= bound).all()), (b, change[b], bound, whole[i])

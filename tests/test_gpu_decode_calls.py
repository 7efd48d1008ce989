"""Calls of the decoding operators that take each of their kernels' forms: sizes of a batch, and inputs that are masked, equal
or rounded."""

import math

import pytest
import torch

import decode_ref as R
from helpers import gpu_available
from test_gpu_decode import World, attend, randn

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


# ---------------------------------------------------------------- beam search

def beam_logits(shape, S, B, V, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(S, B, V, generator=g)
    if shape == "normal":
        return (3 * x).to(dtype)
    if shape == "rounded":
        return torch.round(3 * x).to(dtype)
    if shape == "one lane":  # of a wave's 64, whose 8 consecutive logits are all larger than the others'
        return (x / 8 + 4.0 * (torch.arange(V) // 8 % 64 == 9)).to(dtype)
    kind, count = shape
    rest = {"allowed": -math.inf, "filled": -1.0e4, "above": 0.0}[kind]
    y = torch.full((S, B, V), rest)
    where = torch.rand(S, B, V, generator=g).topk(count).indices if count else torch.zeros(S, B, 0, dtype=torch.long)
    values = torch.randint(1, 4, (S, B, count), generator=g).float() if kind == "above" else x[..., :count]
    return y.scatter(2, where, values).to(dtype)


def beam_scores(S, B, seed):
    return -4 * torch.rand(S, B, generator=torch.Generator().manual_seed(seed))


def best_of(logits, scores, picks):
    """[S][picks] of (score, beam, token) in the order that the header gives, and the smallest distance of two beams' scores
    that follow each other there."""
    x = logits.double()
    v, t = torch.sort(x, dim=2, descending=True, stable=True)
    v, t = v[..., :picks + 1], t[..., :picks + 1]
    v = scores.double()[..., None] + (v - torch.logsumexp(x, 2, keepdim=True))
    found, near = [], math.inf
    for s in range(x.shape[0]):
        # a beam's own are in order; those of several that are equal, of the lower beam first
        c = [(float(a), b, int(i)) for b in range(x.shape[1]) for a, i in zip(v[s, b], t[s, b])]
        c.sort(key=lambda e: (-e[0], e[1]))
        near = min([near] + [a[0] - b[0] for a, b in zip(c[:picks], c[1:picks + 1]) if a[1] != b[1] and math.isfinite(a[0])])
        found.append(c[:picks])
    return found, near


# rows and vocabularies that give a thread 1, 2, 4 and (bf16) 8 vectors of 8 logits
BEAM_SIZES = [(F32, 2, 4, 5003, 8, 1), (F32, 4, 4, 32003, 64, 2), (F32, 4, 4, 60007, 16, 4), (BF16, 2, 4, 5003, 8, 1),
              (BF16, 4, 4, 32003, 5, 2), (BF16, 8, 4, 32003, 8, 4), (BF16, 4, 4, 120_001, 16, 8), (BF16, 4, 4, 120_001, 64, 8)]
BEAM_SHAPES = ["normal", "rounded", "one lane", ("allowed", 4), ("allowed", 12), ("allowed", 60), ("allowed", 200), ("filled", 1),
               ("filled", 12), ("filled", 700), ("above", 0), ("above", 1), ("above", 7), ("above", 63)]


@pytest.mark.parametrize("dtype,S,B,V,picks,vectors", BEAM_SIZES)
@pytest.mark.parametrize("shape", BEAM_SHAPES, ids=str)
def test_beams_of_any_logits(ctx, shape, dtype, S, B, V, picks, vectors):
    """Masked, equal and rounded logits, where few of a wave's vectors stand out or more than there is room for."""
    logits, scores = beam_logits(shape, S, B, V, dtype, V + picks), beam_scores(S, B, 3)
    want, near = best_of(logits, scores, picks)
    assert near > 2.0 ** -19, near  # what the sum of exponentials may be off by, twice
    g = logits.to(DEV)
    search = native.BeamSearch(ctx, g, picks=picks)
    # a list of picks for each stretch of 2048 logits and as many times more as a thread has vectors
    part = 16 + (picks + 1) // 2 * 16
    assert search.workspace_bytes() == S * B * -(-V // (2048 * vectors)) * part
    tokens, parents = (torch.full((S, picks), -5, dtype=torch.int32, device=DEV) for _ in range(2))
    new = torch.full((S, picks), 5.0, device=DEV)
    ws = torch.full((search.workspace_bytes(),), 0xff, dtype=torch.uint8, device=DEV)
    search.select(g, scores.to(DEV), tokens, parents, new, workspace=ws)
    for s in range(S):
        assert list(zip(parents[s].tolist(), tokens[s].tolist())) == [(b, t) for _, b, t in want[s]], s
        for got, (v, _, _) in zip(new[s].tolist(), want[s]):
            assert got == v if math.isinf(v) else abs(got - v) <= 2.0 ** -20 + R.U * abs(v), s


@pytest.mark.parametrize("dtype,S,B,V,picks,vectors", BEAM_SIZES)
def test_beams_without_numbers_of_any_size(ctx, dtype, S, B, V, picks, vectors):
    """Beams of nothing but -inf, with a NaN, with an infinity, without a score, and ended ones, beside others."""
    end = 3
    x, scores = beam_logits("normal", S, B, V, dtype, V), beam_scores(S, B, 4)
    x[0, 0] = -math.inf
    x[0, 1, V - 1] = math.nan
    x[0, 2, 5] = math.inf
    scores[1, 0], scores[1, 1] = -math.inf, math.nan
    ended = torch.zeros(S, B, dtype=torch.int32)
    ended[1, 2] = ended[S - 1, 3] = 1
    x[1, 2] = math.nan  # not looked at
    found = [[] for _ in range(S)]
    for s in range(S):
        for b in range(B):
            v = scores[s, b].double() + torch.log_softmax(x[s, b].double(), 0)
            if ended[s, b]:
                v = torch.full((V,), -math.inf, dtype=torch.float64)
                v[end] = scores[s, b].double()
            if not bool(v.max() > -math.inf):  # of a NaN too
                v = torch.full((V,), -math.inf, dtype=torch.float64)
            a, t = torch.sort(v, descending=True, stable=True)
            found[s] += [(float(p), b, int(i)) for p, i in zip(a[:picks], t[:picks])]
        found[s].sort(key=lambda e: (-e[0], e[1]))
        near = [p[0] - q[0] for p, q in zip(found[s][:picks], found[s][1:]) if p[1] != q[1] and math.isfinite(p[0])]
        assert min(near, default=1) > 2.0 ** -18
    g = x.to(DEV)
    search = native.BeamSearch(ctx, g, picks=picks, end_token=end)
    tokens, parents, done = (torch.full((S, picks), -5, dtype=torch.int32, device=DEV) for _ in range(3))
    new = torch.full((S, picks), 5.0, device=DEV)
    search.select(g, scores.to(DEV), tokens, parents, new, ended=ended.to(DEV), new_ended=done,
                  workspace=torch.full((search.workspace_bytes(),), 0xff, dtype=torch.uint8, device=DEV))
    for s in range(S):
        want = found[s][:picks]
        assert list(zip(parents[s].tolist(), tokens[s].tolist())) == [(b, t) for _, b, t in want], s
        assert done[s].tolist() == [int(t == end or bool(ended[s, b])) for _, b, t in want]
        for got, (v, _, _) in zip(new[s].tolist(), want):
            assert got == v if math.isinf(v) else abs(got - v) <= 2.0 ** -19 + R.U * abs(v), s


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [3000, 8192, 16384])
@pytest.mark.parametrize("case", ["normal", "flat", "steps", "far", "large", "largest"])
def test_beams_sum_of_exponentials(ctx, case, V, dtype):
    """The logarithm of the sum of exponentials is off by less than the header says: a beam's score takes it to nearly 0, of
    which fp32 loses nothing."""
    S = 128  # enough for a thread's most vectors
    g = torch.Generator().manual_seed(V)
    x = torch.randn(S, 1, V, generator=g)
    if case == "flat":
        x = 5 * x.clamp(-1, 1)
    elif case == "steps":  # equal terms below the largest, whose sum is rounded the same way at each step
        x = torch.linspace(-3, 0, S)[:, None, None].expand(S, 1, V).clone()
        x[..., 7] = 0.25
    elif case == "far":
        x = 4 * x - 1000
    elif case == "large":
        x = x + 2.0 ** 21
    elif case == "largest":
        x = torch.where(x > 1, 2.0 ** 29 + 2.0 ** 27, 2.0 ** 20)
    x = x.to(dtype)
    lse, top = torch.logsumexp(x.double(), 2)[:, 0], x.amax(2)[:, 0].double()
    scores = (lse - top).float()
    logits = x.to(DEV)
    search = native.BeamSearch(ctx, logits, picks=1)
    tokens, parents = (torch.empty(S, 1, dtype=torch.int32, device=DEV) for _ in range(2))
    new = torch.empty(S, 1, device=DEV)
    search.select(logits, scores[:, None].to(DEV), tokens, parents, new,
                  workspace=torch.empty(search.workspace_bytes(), dtype=torch.uint8, device=DEV))
    off = new[:, 0].cpu().double() - (scores.double() + (top - lse))
    loose = 2.0 ** -50 * lse.abs()  # of the definition itself, in 64 bits
    limit = 2.0 ** -17 if case in ("large", "largest") else 2.0 ** -19
    assert bool((off.abs() <= limit + loose).all()), float(off.abs().max())


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("L,KV,G,D", [(1, 1, 16, 64), (1, 1, 17, 64), (1, 2, 40, 128), (2, 3, 16, 64), (5, 2, 4, 128), (40, 1, 4, 64),
                                      (150, 2, 1, 128), (33, 1, 2, 64)])
@pytest.mark.parametrize("rotary", [None, 32])
def test_bf16_pages_keep_their_bits(ctx, L, KV, G, D, rotary):
    """bf16 queries over bf16 pages: q' and P are off by 2^-16, as 2^-8 of 2^-8, for any number of rows."""
    n = [L + 300, L, 90 + L]
    w = World(ctx, "bf16", 3, KV, D, 32, 300 + L, BF16, rotary, interleaved=True)
    w.random(1, [0] * 3, n, gain=1.5)
    q = randn(2, 3, L, KV * G, D, dtype=BF16)
    start = [x - L for x in n]
    out = attend(w, q, start=start, causal=True, scale=D ** -0.5, check=False)
    for s in range(3):
        turn = (lambda x, s=s: R.rotary(x[None], [start[s]], rotary, True)[0][0]) if rotary else None
        val, tol = R.attention("bf16", q[s], w.ref.values(s, 0), w.ref.values(s, 1), scale=D ** -0.5, causal=True, start=start[s],
                               turn=turn, operand=2.0 ** -16)
        R.assert_within(out[s], val, tol, f"sequence {s}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("L,KV,G,D,before", [(64, 1, 1, 64, 0), (64, 2, 2, 128, 37), (20, 1, 4, 64, 300), (150, 1, 1, 128, 0), (40, 1, 2, 64, 3000)])
def test_causal_rows_know_only_what_they_see(ctx, kind, L, KV, G, D, before, dtype):
    """Later tokens in other blocks, 2^30 times larger or (8 bits) no numbers: a row before them is the same, bit for bit, and
    as exact as if they were not there."""
    n = before + L
    first = -(-(before + L // 2) // 16) * 16  # a block's first token
    q = randn(2, 1, L, KV * G, D, dtype=dtype)
    results = []
    for gain in (1.0, 2.0 ** 30, 2.0 ** -30, math.nan if kind == "int8" else 5.0):
        w = World(ctx, kind, 1, KV, D, 64, n, dtype, 32)
        w.random(1, [0], [first])
        w.random(5, [first], [n - first], gain=gain)
        out = attend(w, q, start=[before], causal=True, scale=D ** -0.5, check=False)
        results.append(out[0, :first - before].cpu())
    turn = lambda x: R.rotary(x[None], [before], 32, False)[0][0]  # noqa: E731
    val, tol = R.attention(kind, q[0, :first - before], w.ref.values(0, 0, first), w.ref.values(0, 1, first), scale=D ** -0.5,
                           causal=True, start=before, turn=turn)
    for got in results:
        R.assert_within(got, val, tol, "rows before")
        assert torch.equal(got, results[0])


def rows_in(w, q, out, s, first, count, start, keys, scale):
    """Rows first .. of sequence s against the definition."""
    at = start[s] + first
    turn = (lambda x: R.rotary(x[None], [at], w.rotary.c.dim, w.interleaved)[0][0]) if w.rotary else None
    rows = slice(first, first + count)
    operand = 2.0 ** -16 if w.ref.kind == "bf16" and q.dtype == BF16 else None
    val, tol = R.attention(w.ref.kind, q[s, rows], w.ref.values(s, 0, keys[s]), w.ref.values(s, 1, keys[s]), scale=scale, causal=True,
                           start=at, turn=turn, operand=operand)
    R.assert_within(out[s, rows], val, tol, f"sequence {s}, rows from {first}")


# From 64 (sequence, key head) pairs on, workgroups are dealt out to the XCDs pair by pair, and from 512 workgroups of 128
# rows (fp32 of 128 dims: 64) on, each wave has rows of its own; a wave looks up 64 blocks of the table at a time.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("S,KV,G,D,L,n", [(43, 3, 1, 64, 520, 1500), (43, 3, 1, 128, 520, 1500),  # rows of their own, 129 pairs
                                          (4, 2, 4, 64, 2048, 2300),  # rows of their own, 8 pairs
                                          (33, 2, 1, 64, 100, 700), (33, 2, 2, 128, 50, 700)])  # shared rows, 66 pairs
def test_many_rows(ctx, kind, S, KV, G, D, L, n, dtype):
    """Pieces of prompts of large batches, uneven, an empty slot among them."""
    w = World(ctx, kind, S, KV, D, 64, n, dtype, 32, interleaved=True)
    keys = [n - 37 * s % (n - 20) if s != 1 else 0 for s in range(S)]
    rows = [min(L, k) for k in keys]
    start = [k - r for k, r in zip(keys, rows)]
    w.random(1, [0] * S, keys)
    q = randn(2, S, L, KV * G, D, dtype=dtype)
    out = attend(w, q, start=start, query_lengths=rows, causal=True, scale=D ** -0.5, check=False)
    for s in (0, S // 2, S - 1):
        for first in (0, rows[s] // 2, max(rows[s] - 9, 0)):
            rows_in(w, q, out, s, first, min(9, rows[s] - first), start, keys, D ** -0.5)
    for s in range(S):
        assert bool((out[s, rows[s]:] == 0).all()) and bool(out[s].isfinite().all()), s


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_one_piece_of_many_keys(ctx, kind, D, dtype):
    """Single tokens of 64 sequences of 4 key heads, whose keys are not cut: three sequences are long."""
    S, KV, n = 64, 4, 4700
    w = World(ctx, kind, S, KV, D, 64, n, dtype, 32)
    keys = [7] * S
    w.random(1, [0] * S, keys)
    for i, s in enumerate((0, 30, 63)):
        keys[s] = n - 300 * i
        k, v = (randn(10 * i + j, 1, keys[s], KV, D, dtype=dtype) for j in (3, 4))
        w.cache.tokens(w.table[s:s + 1].contiguous(), k.to(DEV), v.to(DEV), rotary=w.rotary).append(k.to(DEV), v.to(DEV))
        w.ref.append(s, 0, R.turn32(k[0].float(), w.rotary.table.cpu(), 0, False), v[0].float())
    q = randn(2, S, 1, KV, D, dtype=dtype)
    g = q.to(DEV)
    assert w.cache.queries(w.table, g, g, most_keys=n).workspace_bytes() == 16  # no pieces to join
    start = [x - 1 for x in keys]
    out = attend(w, q, start=start, keys=keys, scale=D ** -0.5, check=False)
    for s in (0, 1, 30, 62, 63):
        rows_in(w, q, out, s, 0, 1, start, keys, D ** -0.5)

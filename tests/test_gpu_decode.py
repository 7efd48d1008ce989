"""Rotary positions, the paged cache with its attention, and beam search on the GPU against their definitions."""

import math

import pytest
import torch

import decode_ref as R
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


def randn(seed, *shape, dtype=F32):
    g = torch.Generator()
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype)


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def buffer(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=DEV).fill_(0xff)


# ---------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S,L,H,D,dim", [(1, 1, 1, 2, 2), (2, 5, 3, 64, 64), (3, 17, 2, 80, 40), (1, 33, 7, 96, 24),
                                         (2, 9, 1, 67, 6), (1, 300, 40, 128, 128), (2, 3, 2, 512, 256), (1, 7, 3, 11, 10)])
def test_rotary(ctx, S, L, H, D, dim, dtype, interleaved, backward):
    x = randn(S + L + D, S, L, H, D, dtype=dtype)
    start = [0, 7, 1000][:S]
    r = native.Rotary(ctx, 1000 + L, dim, interleaved=interleaved)
    y = torch.empty(S, L, H, D, dtype=dtype, device=DEV).fill_(math.nan)
    r.apply(x.to(DEV), y, start=ints(start), backward=backward)
    val, tol = R.rotary(x, start, dim, interleaved, backward)
    R.assert_within(y, val, tol, "y")
    here = x.to(DEV)
    r.apply(here, here, start=ints(start), backward=backward)  # in place
    assert torch.equal(here, y)


@pytest.mark.parametrize("angles", [dict(base=500000.0), dict(factor=4.0), dict(factor=8.0, original=8192, low=1.0, high=32.0,
                                                                               magnitude=1.21),
                                    dict(factor=2.0, original=100, low=0.5, high=2.0)], ids=str)
def test_rotary_scaled_far(ctx, angles):
    x = randn(1, 2, 3, 2, 64)
    r = native.Rotary(ctx, 200_003, 64, **angles)
    y = torch.empty_like(x, device=DEV)
    start = [200_000, 131_071]
    r.apply(x.to(DEV), y, start=ints(start))
    val, tol = R.rotary(x, start, 64, False, **angles)
    R.assert_within(y, val, tol, "y")


def test_rotary_strides(ctx):
    """Slices of one projection, rows before heads, and places between rows left as they were."""
    qkv = randn(3, 2, 6, 3, 4, 64, dtype=BF16)
    g = qkv.to(DEV)
    wide = torch.full((2, 4, 6, 100), 5.0, dtype=BF16, device=DEV)
    y = wide.transpose(1, 2)[..., 3:67]  # [S][L][H][64], rows inside heads, from an odd element on
    r = native.Rotary(ctx, 6, 48, interleaved=True)
    r.apply(g[:, :, 1], y)
    val, tol = R.rotary(qkv[:, :, 1], [0, 0], 48, True)
    R.assert_within(y, val, tol, "y")
    assert bool((wide[..., :3] == 5).all()) and bool((wide[..., 67:] == 5).all())
    r.apply(g[:, :, 0], g[:, :, 0])
    val, tol = R.rotary(qkv[:, :, 0], [0, 0], 48, True)
    R.assert_within(g[:, :, 0], val, tol, "in place")
    assert torch.equal(g[:, :, 1:].cpu(), qkv[:, :, 1:])


def test_rotary_gradient(ctx):
    """backward is the transpose: against differences of the forward's definition, and <y, Rx> = <R^T y, x>."""
    x, dy = randn(5, 1, 4, 2, 32).to(DEV), randn(6, 1, 4, 2, 32).to(DEV)
    r = native.Rotary(ctx, 4, 32, factor=2.0, original=16, low=0.1, high=1.0, magnitude=1.3)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    r.apply(x, y)
    r.apply(dy, dx, backward=True)
    a, b = (dy.double() * y.double()).sum(), (dx.double() * x.double()).sum()
    assert abs(a - b) <= 8 * R.U * (dy.double().abs() * 2 * 1.3 * x.double().abs().amax()).sum()
    z = torch.empty_like(x)
    for i in range(0, x.numel(), 37):
        xx = x.clone()
        xx.view(-1)[i] += 1  # linear: a whole step
        r.apply(xx, z)
        d = ((z.double() - y.double()) * dy.double()).sum()
        assert abs(d - dx.view(-1)[i].double()) <= 64 * R.U * (z.abs().amax() + 1) * dy.double().abs().sum()


def test_rotary_positions_beyond_the_table(ctx):
    x = randn(7, 3, 4, 1, 8).to(DEV)
    y = torch.empty_like(x)
    native.Rotary(ctx, 6, 4).apply(x, y, start=ints([0, 4, -2]))
    y = y.cpu()
    assert bool(y[0].isfinite().all()) and bool(y[1, :2].isfinite().all()) and bool(y[2, 2:].isfinite().all())
    assert bool(y[1, 2:, :, :4].isnan().all()) and bool(y[2, :2, :, :4].isnan().all())
    assert torch.equal(y[..., 4:], x.cpu()[..., 4:])


def test_rotary_nothing(ctx):
    r = native.Rotary(ctx, 4, 4)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8)):
        x = torch.empty(shape, device=DEV)
        r.apply(x, x)


# ---------------------------------------------------------------- the cache

class World:
    """A cache on the GPU beside its definition; sequences' pages scattered over the pool."""

    def __init__(self, ctx, kind, S, KV, D, page, capacity, dtype, rotary=None, interleaved=False, seed=0):
        self.ctx, self.S, self.KV, self.D, self.dtype = ctx, S, KV, D, dtype
        each = -(-capacity // page)
        g = torch.Generator()
        g.manual_seed(seed)
        ids = torch.randperm(S * each + 3, generator=g)
        self.table = ids[:S * each].view(S, each).int().to(DEV).contiguous()
        self.cache = native.PagedCache(ctx, kind, kv_heads=KV, head_dim=D, page_tokens=page, pages=S * each + 3)
        self.cache.pool.fill_(0xff)  # NaN as bf16 and as scales
        self.ref = R.Cache(kind, S, KV, D)
        self.rotary = native.Rotary(ctx, capacity, rotary, interleaved=interleaved) if rotary else None
        self.interleaved = interleaved

    def append(self, k, v, start, lengths):
        self.cache.tokens(self.table, k.to(DEV), v.to(DEV), start=ints(start), lengths=ints(lengths),
                          rotary=self.rotary).append(k.to(DEV), v.to(DEV))
        for s in range(self.S):
            kk = k[s, :lengths[s]].float()
            if self.rotary:
                kk = R.turn32(kk, self.rotary.table.cpu(), start[s], self.interleaved)
            self.ref.append(s, start[s], kk, v[s, :lengths[s]].float())

    def random(self, seed, start, lengths, gain=1.0):
        n = max(max(lengths), 1)
        k, v = (gain * randn(seed + i, self.S, n, self.KV, self.D) for i in (0, 1))
        self.append(k.to(self.dtype), v.to(self.dtype), start, lengths)

    def read(self, start, lengths, length):
        k, v = (torch.full((self.S, length, self.KV, self.D), 9.0, dtype=self.dtype, device=DEV) for _ in "kv")
        self.cache.tokens(self.table, k, v, start=ints(start), lengths=ints(lengths)).read(k, v)
        return k, v

    def check(self):
        n = max(self.ref.n)
        got = self.read([0] * self.S, self.ref.n, n + 3)
        for s in range(self.S):
            for part in (0, 1):
                want = self.ref.values(s, part).to(self.dtype)
                here = got[part][s].cpu()
                assert torch.equal(here[:self.ref.n[s]], want), (s, "kv"[part])
                assert bool((here[self.ref.n[s]:] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("KV,D,page,rotary,interleaved", [(1, 64, 16, None, False), (3, 64, 48, 64, True), (2, 128, 32, 128, False),
                                                          (4, 128, 16, 48, False), (2, 64, 4096, 32, True)])
def test_append_and_read(ctx, kind, KV, D, page, rotary, interleaved, dtype):
    """Prompts of uneven lengths, then tokens by ones and by several, over block and page ends; what comes back is what the
    definition holds, bit for bit."""
    S = 4
    w = World(ctx, kind, S, KV, D, page, 200, dtype, rotary, interleaved)
    n = [0, 1, 16, 37]
    w.random(1, [0] * S, n)
    w.check()
    for i, step in enumerate(([1, 1, 1, 1], [1, 0, 1, 1], [5, 17, 2, 30], [1, 1, 1, 1], [40, 3, 64, 1])):
        w.random(10 + i, n, step, gain=0.5 + i)  # growing: earlier tokens of a block are rescaled
        n = [a + b for a, b in zip(n, step)]
        w.check()
    # back to an earlier position: what was behind it in its block is lost, tokens after that block stay
    back = [max(0, x - 3) for x in n]
    w.random(50, back, [1] * S)
    w.check()


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_read_in_part(ctx, kind):
    w = World(ctx, kind, 2, 2, 64, 32, 100, BF16)
    w.random(3, [0, 0], [90, 50])
    start, length = [13, 45], 40
    k, v = w.read(start, [40, 9], length)
    for s, (a, n) in enumerate(zip(start, (40, 5))):
        assert torch.equal(k[s, :n].cpu(), w.ref.values(s, 0)[a:a + n].bfloat16())
        assert torch.equal(v[s, :n].cpu(), w.ref.values(s, 1)[a:a + n].bfloat16())
    assert bool((k[1, 9:] == 0).all()) and bool((v[1, 9:] == 0).all())
    only = torch.empty(2, length, 2, 64, dtype=BF16, device=DEV)
    t = w.cache.tokens(w.table, only, only, start=ints(start), lengths=ints([40, 9]))
    t.read(None, only)
    assert torch.equal(only, v)
    t.read(only, None)
    assert torch.equal(only, k)


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_slices_and_what_is_not_there(ctx, kind):
    """k and v as slices of one projection; entries that are no page, tokens beyond the table and starts below 0."""
    S, KV, D, page = 3, 2, 64, 16
    cache = native.PagedCache(ctx, kind, kv_heads=KV, head_dim=D, page_tokens=page, pages=4)
    cache.pool.fill_(0x7f)
    table = ints([[0, -1], [1, 99], [2, 3]])
    qkv = randn(1, S, 40, 5, KV, D, dtype=BF16).to(DEV)
    k, v = qkv[:, :, 1], qkv[:, :, 3]
    cache.tokens(table, k, v, start=ints([0, 4, -5])).append(k, v)  # sequence 2: from 0 on, 40 tokens for 32 places
    before = cache.pool.clone()
    out = torch.full_like(qkv, 7.0)
    cache.tokens(table, out[:, :, 0], out[:, :, 2], start=ints([0, 4, -5])).read(out[:, :, 0], out[:, :, 2])
    half = 0.51 * float(qkv.float().abs().amax()) / 127 if kind == "int8" else 0.0
    for i, x in ((0, k), (2, v)):
        held = [(0, 16), (0, 12), (0, 32)]
        for s, (a, b) in enumerate(held):
            want = x[s, a:b].float()
            if kind == "int8" and s == 1:  # appended behind 4 tokens of what was there: a scale of 3.4e38, beside which these are 0
                want = torch.zeros_like(want)
            off = (out[s, a:b, i].float() - want).abs()
            assert bool((off <= half + 2.0 ** -8 * want.abs() * (kind == "int8")).all()), (s, i)
            assert bool((out[s, b:, i] == 0).all())
    assert bool((out[:, :, [1, 3, 4]] == 7).all()) and torch.equal(before, cache.pool)
    # far beyond the table: nothing is touched
    cache.tokens(table, k, v, start=ints([1000, 2 ** 31 - 1, 2 ** 30])).append(k, v)
    assert torch.equal(before, cache.pool)


def test_numbers_beyond_the_scale(ctx):
    """A block of zeros, of the smallest numbers, of the largest, and with an infinity or a NaN, which all of the block's
    head becomes; the next block is as it was."""
    KV, D = 2, 64
    for x, want in ((0.0, 0.0), (1e-38, 0.0), (3.3e38, 3.3e38), (math.inf, math.nan), (math.nan, math.nan)):
        w = World(ctx, "int8", 1, KV, D, 16, 32, F32)
        k = torch.ones(1, 20, KV, D)
        k[0, :16] = 0
        k[0, 3, 1, 5] = x
        w.cache.tokens(w.table, k.to(DEV), k.to(DEV)).append(k.to(DEV), k.to(DEV))
        for t in w.read([0], [20], 20):
            t = t.cpu()
            assert bool((t[0, :16, 0] == 0).all()) and bool(((t[0, 16:] - 1).abs() <= 2 * R.U).all())
            if math.isnan(want):
                assert bool(t[0, :16, 1].isnan().all())
            else:
                assert abs(float(t[0, 3, 1, 5]) - want) <= 4 * R.U * abs(want) + 2.0 ** -101
    # a token after it in the same block does not bring it back
    w = World(ctx, "int8", 1, 1, 64, 16, 32, F32)
    k = torch.full((1, 1, 1, 64), math.nan, device=DEV)
    w.cache.tokens(w.table, k, k).append(k, k)
    w.cache.tokens(w.table, k, k, start=ints([1])).append(torch.ones_like(k), torch.ones_like(k))
    assert all(bool(t[0, :2].isnan().all()) for t in w.read([0], [2], 2))
    # what was left in the block's place from before is not looked at
    w.cache.tokens(w.table, k, k, start=ints([0])).append(torch.ones_like(k), torch.ones_like(k))
    assert all(bool((t[0, 0] - 1).abs().amax() <= 2 * R.U) for t in w.read([0], [1], 1))


# ---------------------------------------------------------------- attention

def attend(w, q, *, start, keys=None, query_lengths=None, most=None, check=True, **more):
    """The cache's attention and its definition over the values that the cache holds."""
    S, L, H, D = q.shape
    keys = w.ref.n if keys is None else keys
    most = max(max(keys), 1) if most is None else most
    g, out = q.to(DEV), torch.full(q.shape, 3.0, dtype=q.dtype, device=DEV)
    plan = w.cache.queries(w.table, g, out, most_keys=most, key_lengths=ints(keys), query_start=ints(start),
                           query_lengths=ints(query_lengths) if query_lengths else None, rotary=w.rotary, **more)
    ws = buffer(plan.workspace_bytes())
    plan.forward(g, out, workspace=ws)
    again = torch.empty_like(out)
    ws.fill_(0)
    plan.forward(g, again, workspace=ws)
    assert torch.equal(out.view(torch.uint8), again.view(torch.uint8))  # equal calls, equal bits
    if check:
        kind = w.ref.kind
        for s in range(S):
            n = max(0, min(keys[s], most))
            m = query_lengths[s] if query_lengths else L
            turn = None
            if w.rotary:
                turn = lambda x, s=s: R.rotary(x[None], [start[s]], w.rotary.c.dim, w.interleaved)[0][0]  # noqa: E731
            val, tol = R.attention(kind, q[s], w.ref.values(s, 0, n), w.ref.values(s, 1, n), start=start[s], turn=turn, **more)
            val[m:], tol[m:] = 0, 0
            R.assert_within(out[s], val, tol, f"sequence {s}")
    return out


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("KV,G,D,page,rotary", [(1, 1, 64, 16, 64), (2, 4, 64, 64, 32), (2, 3, 128, 48, 128), (1, 16, 128, 32, None),
                                                (1, 24, 64, 16, None)])
def test_single_tokens(ctx, kind, KV, G, D, page, rotary, dtype):
    """Steps of decoding over caches of every length's end: none, one, within and at blocks, steps and pages."""
    n = [0, 1, 15, 16, 17, 63, 64, 65, 129, 300]
    w = World(ctx, kind, len(n), KV, D, page, 320, dtype, rotary, interleaved=bool(page == 64))
    w.random(1, [0] * len(n), n, gain=1.5)
    q = randn(2, len(n), 1, KV * G, D, dtype=dtype)
    out = attend(w, q, start=[max(x - 1, 0) for x in n], scale=D ** -0.5)
    assert bool((out[0] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("L,KV,G,D", [(2, 1, 1, 64), (5, 2, 4, 64), (33, 2, 2, 128), (70, 1, 4, 64), (130, 2, 1, 128), (300, 1, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens(ctx, kind, L, KV, G, D, causal, dtype):
    """Pieces of prompts after what is there, uneven, with padded rows and an empty slot; rows before the first key."""
    n = [L, L + 40, 200 + L, 0, 90]
    w = World(ctx, kind, 5, KV, D, 32, 600, dtype, 32, interleaved=True)
    w.random(4, [0] * 5, n)
    q = randn(5, 5, L, KV * G, D, dtype=dtype)
    attend(w, q, start=[0, 40, 200, 0, 90 - min(L, 90)], query_lengths=[L, max(L - 7, 1), L, 0, min(L, 90)], causal=causal,
           scale=D ** -0.5)
    if causal:  # queries before all keys, and far behind them
        w.rotary = None
        out = attend(w, q, start=[-3, -10 * L, 10 ** 6, 0, 5], causal=True, scale=D ** -0.5)
        assert bool((out[0, :min(3, L)] == 0).all()) and bool((out[1] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("L,KV,G,D,n", [(1, 1, 8, 64, 5000), (1, 2, 2, 128, 3001), (3, 1, 8, 128, 2500), (200, 1, 1, 64, 3000),
                                        (160, 1, 2, 128, 2111)])
def test_keys_in_pieces(ctx, kind, L, KV, G, D, n, dtype):
    """Long caches of few sequences, whose keys are cut into pieces that are joined; one much shorter, whose later pieces
    are empty."""
    lengths = [n, 700, 40 + L]
    w = World(ctx, kind, 3, KV, D, 64, n, dtype, 64)
    w.random(6, [0] * 3, lengths)
    # keys that stand out late, so that the maximum moves from piece to piece
    w.random(8, [n - 40, 600, 10], [5, 5, 5], gain=3.0)
    w.random(9, [n - 35, 605, 15], [35, 95, 25 + L])
    q = randn(7, 3, L, KV * G, D, dtype=dtype)
    attend(w, q, start=[x - L for x in lengths], causal=L > 1, scale=1.3 * D ** -0.5)


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_blocks_of_other_sizes(ctx, kind):
    """Blocks whose keys and values are larger or smaller than others' by many powers of two; queries of any size; a
    negative scale, and none."""
    w = World(ctx, kind, 2, 1, 64, 16, 400, F32)
    for i, gain in enumerate((1.0, 1e-20, 1e6, 1e-3, 1.0, 30.0)):
        w.random(20 + i, [32 * i] * 2, [32, 32], gain=gain)
    q = randn(1, 2, 1, 4, 64)
    q[0, 0, 1] *= 1e-6
    q[0, 0, 2] *= 1e-30
    q[0, 0, 3] = 0
    q[1] *= 1e-7
    for scale in (0.125, -0.125, 0.0, 1e-8):
        attend(w, q, start=[0, 0], scale=scale)


@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("L", [1, 40, 140])
def test_what_lies_behind_the_keys(ctx, kind, L):
    """Tokens from a sequence's key length on change nothing, NaN in bf16 among them; nor do pages that are not there, whose
    tokens no query sees."""
    w = World(ctx, kind, 2, 1, 64, 32, 256, BF16)
    w.random(1, [0, 0], [200, 200])
    q = randn(2, 2, L, 2, 64, dtype=BF16)
    keys = [77, 150]
    a = attend(w, q, start=[0, 0], keys=keys, scale=0.125)
    for s, n in enumerate(keys):
        bad = torch.full((2, 40, 1, 64), math.nan if kind == "bf16" else 1.0, dtype=BF16, device=DEV)
        rows = [0, 0]
        rows[s] = 40
        w.cache.tokens(w.table, bad, bad, start=ints([x + (0 if kind == "bf16" else -x % 16) for x in keys]), lengths=ints(rows)).append(bad, bad)
    b = attend(w, q, start=[0, 0], keys=keys, scale=0.125, check=False)
    assert torch.equal(a, b)
    # most_keys below the lengths
    attend(w, q, start=[0, 0], keys=keys, most=60, scale=0.125)
    # sequence 0's second page (tokens 32 to 63) is none
    w.table[0, 1] = -7
    c = attend(w, q, start=[0, 0], keys=keys, scale=0.125, check=False)
    assert torch.equal(b[1], c[1])
    there = list(range(32)) + list(range(64, 77))
    val, tol = R.attention(kind, q[0], w.ref.values(0, 0, 77)[there], w.ref.values(0, 1, 77)[there], scale=0.125)
    R.assert_within(c[0], val, tol, "without a page")
    w.table.fill_(10 ** 6)
    assert bool((attend(w, q, start=[0, 0], keys=keys, scale=0.125, check=False) == 0).all())


def test_numbers_that_are_none(ctx):
    """A NaN or infinity in a query stays in its row; a block that holds one is one for the rows that see it, and for no
    other sequence."""
    for kind in ("int8", "bf16"):
        w = World(ctx, kind, 2, 1, 64, 16, 64, F32)
        w.random(1, [0, 0], [40, 40])
        q = randn(2, 2, 3, 2, 64)
        clean = attend(w, q, start=[0, 0], scale=0.125)
        q[0, 1, 0, 3] = math.nan
        q[1, 2, 1, 3] = math.inf
        out = attend(w, q, start=[0, 0], scale=0.125, check=False)
        touched = torch.zeros(2, 3, 2, dtype=torch.bool)
        touched[0, 1, 0] = touched[1, 2, 1] = True
        assert torch.equal(out.cpu()[~touched], clean.cpu()[~touched])
        assert bool(out.cpu()[0, 1, 0].isnan().all()) and bool(out.cpu()[1, 2, 1].isnan().any())
        bad = torch.full((2, 1, 1, 64), math.nan, device=DEV)
        w.cache.tokens(w.table, bad, bad, start=ints([40, 0]), lengths=ints([1, 0])).append(bad, bad)
        q = randn(2, 2, 3, 2, 64)
        out = attend(w, q, start=[0, 0], keys=[41, 40], scale=0.125, check=False)
        assert bool(out[0].isnan().all()) and torch.equal(out[1], clean[1])


@pytest.mark.parametrize("kind", ["int8", "bf16"])
def test_nothing_to_attend_to(ctx, kind):
    """No keys for anybody, no pages in the table, no rows, no sequences; key lengths below 0 and beyond the table."""
    w = World(ctx, kind, 2, 1, 64, 16, 48, F32)
    w.random(1, [0, 0], [48, 20])
    q = randn(2, 2, 3, 2, 64)
    assert bool((attend(w, q, start=[0, 0], most=0, keys=[40, 20], scale=0.125, check=False) == 0).all())
    out = attend(w, q, start=[0, 0], keys=[-4, 10 ** 9], most=10 ** 6, scale=0.125, check=False)
    assert bool((out[0] == 0).all())
    # 48 tokens, of which 28 were never appended: what the pool began with, of int8 scales that are no numbers, and the last
    # block of the first 20 ends in zeros
    assert bool(out[1].isnan().all())
    for table in (w.table[:, :0].contiguous(), w.table[:0]):
        S = table.shape[0]
        x, o = q[:S].to(DEV), torch.full((S, 3, 2, 64), 7.0, device=DEV)
        p = w.cache.queries(table, x, o, most_keys=30)
        p.forward(x, o, workspace=buffer(p.workspace_bytes()))
        assert bool((o == 0).all())
        k = torch.ones(S, 5, 1, 64, device=DEV)
        before = w.cache.pool.clone()
        w.cache.tokens(table, k, k).append(k, k)
        assert torch.equal(before, w.cache.pool)
        w.cache.tokens(table, k, k).read(k, None)
        assert bool((k == 0).all())
    x = torch.empty(2, 0, 2, 64, device=DEV)
    p = w.cache.queries(w.table, x, x, most_keys=30)
    p.forward(x, x, workspace=buffer(p.workspace_bytes()))


def test_attention_strides_and_in_place(ctx):
    """Queries as a slice of a projection, out in their place, and out with heads outside rows."""
    w = World(ctx, "int8", 2, 2, 64, 16, 200, BF16, 64)
    w.random(1, [0, 0], [150, 99])
    qkv = randn(2, 2, 3, 8, 64, dtype=BF16)
    q = qkv[:, :, 1:5]
    want = attend(w, q.contiguous(), start=[147, 96], causal=True, scale=0.125)
    g = qkv.to(DEV)
    plan = lambda out: w.cache.queries(w.table, g[:, :, 1:5], out, most_keys=200, causal=True, key_lengths=ints([150, 99]),  # noqa: E731
                                       query_start=ints([147, 96]), rotary=w.rotary)
    turned = torch.empty(2, 4, 3, 64, dtype=BF16, device=DEV).transpose(1, 2)
    for out in (turned, g[:, :, 1:5]):
        p = plan(out)
        p.forward(g[:, :, 1:5], out, workspace=buffer(p.workspace_bytes()))
        R.assert_within(out, want.double().cpu(), 2.1 * R.HALF[BF16] * want.double().cpu().abs() + 2.0 ** -9, "out")
    assert torch.equal(g[:, :, 5:].cpu(), qkv[:, :, 5:]) and torch.equal(g[:, :, 0].cpu(), qkv[:, :, 0])


def test_pool_beyond_32_bits(ctx):
    """Pages more than 4 GB apart."""
    page, KV, D = 4096, 8, 128
    pages = 700  # of 8.4 MB each
    cache = native.PagedCache(ctx, "int8", kv_heads=KV, head_dim=D, page_tokens=page, pages=pages)
    assert cache.pool.numel() > 5 << 30
    table = ints([[pages - 1], [0]])
    k, v = randn(1, 2, 33, KV, D, dtype=BF16).to(DEV), randn(2, 2, 33, KV, D, dtype=BF16).to(DEV)
    cache.tokens(table, k, v).append(k, v)
    q = randn(3, 2, 1, KV, D, dtype=BF16)
    out = torch.empty(2, 1, KV, D, dtype=BF16, device=DEV)
    p = cache.queries(table, q.to(DEV), out, most_keys=33, scale=D ** -0.5)
    p.forward(q.to(DEV), out, workspace=buffer(p.workspace_bytes()))
    ref = R.Cache("int8", 2, KV, D)
    for s in range(2):
        ref.append(s, 0, k[s].float().cpu(), v[s].float().cpu())
        val, tol = R.attention("int8", q[s], ref.values(s, 0), ref.values(s, 1), scale=D ** -0.5)
        R.assert_within(out[s], val, tol, f"sequence {s}")


# ---------------------------------------------------------------- beam search

def select(ctx, logits, scores, picks, end_token=-1, ended=None):
    S, B, V = logits.shape
    g = logits.to(DEV) if not logits.is_cuda else logits
    search = native.BeamSearch(ctx, g, picks=picks, end_token=end_token)
    tokens, parents, done = (torch.full((S, picks), -5, dtype=torch.int32, device=DEV) for _ in range(3))
    new = torch.full((S, picks), 5.0, device=DEV)
    search.select(g, scores.to(DEV), tokens, parents, new, ended=None if ended is None else ended.int().to(DEV), new_ended=done,
                  workspace=buffer(search.workspace_bytes()))
    return tokens.cpu(), parents.cpu(), new.cpu(), done.cpu()


def check_beams(ctx, logits, scores, picks, end_token=-1, ended=None):
    tokens, parents, new, done = select(ctx, logits, scores, picks, end_token, ended)
    # a sum of exponentials of 32 terms a lane and its logarithm: 2^-20 is far above what that is off by
    for s in range(logits.shape[0]):
        want, near = R.beams(logits[s], scores[s], picks, end_token, None if ended is None else ended[s])
        assert near > 2.0 ** -19, f"sequence {s}: the inputs do not tell an order ({near})"
        assert [(int(p), int(t)) for p, t in zip(parents[s], tokens[s])] == [(b, t) for _, b, t in want], s
        for i, (v, b, t) in enumerate(want):
            if math.isinf(v):
                assert float(new[s, i]) == v
            else:
                assert abs(float(new[s, i]) - v) <= 2.0 ** -20 + R.U * abs(v), (s, i)
            assert int(done[s, i]) == int(t == end_token or (ended is not None and bool(ended[s, b])))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("S,B,V,picks", [(1, 1, 1, 1), (1, 2, 1, 2), (2, 3, 2, 5), (1, 4, 63, 64), (3, 4, 1000, 4), (2, 5, 8191, 10),
                                         (1, 2, 8193, 7), (1, 3, 16385, 3), (2, 2, 33001, 64), (1, 2, 70001, 16), (1, 64, 100, 64),
                                         (1, 1, 200_003, 1)])
def test_beams(ctx, S, B, V, picks, dtype):
    logits = (3 * randn(S + V, S, B, V)).to(dtype)
    check_beams(ctx, logits, -randn(9, S, B).abs(), picks)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beams_ended(ctx, dtype):
    logits = (2 * randn(1, 4, 3, 500)).to(dtype)
    logits[0, 1] = math.nan  # of an ended beam: not looked at
    ended = torch.tensor([[0, 1, 0], [1, 1, 1], [0, 0, 0], [1, 0, 1]])
    for end in (0, 7, 499):
        check_beams(ctx, logits, -1 - randn(2, 4, 3).abs(), 6, end, ended)
        check_beams(ctx, logits[1:], -1 - randn(2, 3, 3).abs(), 6, end)


@pytest.mark.parametrize("V", [700, 40000])
def test_beams_alike(ctx, V):
    """Equal logits: the lowest token first; equal beams: the lowest beam; all of a wave's alike, so that none stands out."""
    for x in (torch.zeros(1, 2, V), torch.full((1, 2, V), -0.0), torch.full((1, 2, V), 1e-30)):
        tokens, parents, new, _ = select(ctx, x, torch.tensor([[-1.0, -1.0]]), 9)
        assert tokens[0].tolist() == list(range(9)) and parents[0].tolist() == [0] * 9
        assert bool(((new + 1 + math.log(V)).abs() < 1e-5).all())
    x = torch.zeros(1, 1, V)
    x[0, 0, 1::2] = -0.0  # equal to 0
    assert select(ctx, x, torch.zeros(1, 1), 6)[0][0].tolist() == list(range(6))
    x = torch.zeros(1, 1, V)
    x[0, 0, V - 3:] = 1.0
    x[0, 0, 600] = 1.0
    assert select(ctx, x, torch.zeros(1, 1), 7)[0][0].tolist() == [600, V - 3, V - 2, V - 1, 0, 1, 2]


def test_beams_in_one_lane(ctx):
    """Rising, falling and comb-shaped logits, whose largest are all in a few lanes' registers."""
    V = 65536
    t = torch.arange(V, dtype=torch.float32)
    for x in (t / V, -t / V, (t % 64 == 5) * 4.0 + t / V, (t // 8 % 1024 == 77) * 4.0 - t / V, (t // 8 % 64 == 9) * 4.0 + t / V):
        want = torch.sort(x, descending=True, stable=True).indices[:64].tolist()
        assert select(ctx, x.view(1, 1, V), torch.zeros(1, 1), 64)[0][0].tolist() == want


def test_beams_without_numbers(ctx):
    """-inf logits and scores, NaN and +inf: candidates of -inf in order, behind all others."""
    x = randn(3, 6, 2, 300)
    x[0, 0] = -math.inf
    x[1, 1, 7] = math.nan
    x[2, 0, 9] = math.inf
    x[3, :, 2:] = -math.inf
    scores = -torch.ones(6, 2)
    scores[0, 1] = -2.5
    scores[4] = torch.tensor([-math.inf, -1.0])
    scores[5] = torch.tensor([math.nan, math.inf])
    tokens, parents, new, _ = select(ctx, x, scores, 8)
    for s in range(6):
        want, _ = R.beams(x[s], scores[s], 8)
        assert [(int(p), int(t)) for p, t in zip(parents[s], tokens[s])] == [(b, t) for _, b, t in want], s
        assert [math.isinf(float(v)) for v in new[s]] == [math.isinf(v) for v, _, _ in want]
    assert tokens[5].tolist() == list(range(8)) and parents[5].tolist() == [0] * 8


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("top", [1.0e4, 1.7e7, 5.4e8, 1.07e9, 1.08e9, 2.2e9, 3.3e38, -1.7e7, -1.07e9, -3.3e38])
def test_beams_large_logits(ctx, top, dtype):
    """Logits around a large number: the largest one several times, the next numbers of the type, ones far below, -0."""
    x = torch.full((1, 2, 5000), -0.0 if top > 0 else 1.02 * top)
    up = torch.tensor(top).to(dtype)
    for beam, alike in ((0, 3), (1, 4)):
        v = up.clone()
        for token in (4990, 17, 2500):
            x[0, beam, token] = float(v)
            v = torch.nextafter(v, torch.tensor(-math.inf, dtype=dtype))
        x[0, beam, 100:100 + alike] = float(up)
    check_beams(ctx, x.to(dtype), torch.tensor([[-1.0, -1.5]]), 6)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V", [200, 5000, 40000])
@pytest.mark.parametrize("allowed,picks", [(0, 64), (3, 64), (3, 5), (40, 64), (64, 64), (300, 64), (1000, 16)])
def test_beams_few_tokens_allowed(ctx, V, allowed, picks, dtype):
    """All logits but a few -inf, in one stretch or all over: the others fill up from the lowest token."""
    g = torch.Generator().manual_seed(V + allowed)
    allowed = min(allowed, V)
    for where in (torch.randperm(V, generator=g)[:allowed], torch.arange(V - allowed, V)):
        x = torch.full((1, 2, V), -math.inf)
        # of bf16's values, each beam's apart from the other's
        x[0, 0, where] = (torch.randperm(allowed, generator=g) / 64).float()
        x[0, 1, where] = (torch.randperm(allowed, generator=g) / 64).float()
        x = x.to(dtype)
        scores = torch.tensor([[-1.0, -1.3]])
        tokens, parents, new, _ = select(ctx, x, scores, picks)
        want, near = R.beams(x[0], scores[0], picks)
        assert near > 2.0 ** -19, near
        assert [(int(p), int(t)) for p, t in zip(parents[0], tokens[0])] == [(b, t) for _, b, t in want]
        assert [math.isinf(float(v)) for v in new[0]] == [math.isinf(v) for v, _, _ in want]


def test_beams_many_lists(ctx):
    """More lists of candidates than are compared at one place: sorted one part after the other."""
    B, V, picks = 64, 140_003, 64
    x = randn(11, 1, B, V)
    scores = -randn(12, 1, B).abs() / 4
    s = (torch.log_softmax(x[0].double(), -1) + scores[0].double()[:, None]).flatten()
    best = s.topk(picks + 1)
    assert float((best.values[:-1] - best.values[1:]).min()) > 2.0 ** -19
    for logits in (x, x.to(DEV)[:, :, :]):
        tokens, parents, new, _ = select(ctx, logits, scores, picks)
        assert (parents[0].long() * V + tokens[0].long()).tolist() == best.indices[:picks].tolist()
        assert float((new[0].double() - best.values[:picks]).abs().max()) <= 2.0 ** -20 + R.U * float(best.values.abs().max())


def test_beams_strides(ctx):
    wide = randn(4, 3, 5, 1003).to(DEV)
    x = wide[:, 1:4, 1:1000]
    check_beams(ctx, x.cpu(), -randn(1, 3, 3).abs(), 4)
    a = select(ctx, x, -randn(1, 3, 3).abs(), 4)
    b = select(ctx, x.contiguous(), -randn(1, 3, 3).abs(), 4)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


# ---------------------------------------------------------------- beams' tables

@pytest.mark.parametrize("kind", ["int8", "bf16"])
@pytest.mark.parametrize("page,length", [(16, 16), (16, 5), (16, 33), (64, 75), (48, 100), (64, 0), (32, 96)])
def test_reorder(ctx, kind, page, length):
    G, B, KV, D = 2, 4, 2, 64
    w = World(ctx, kind, G * B, KV, D, page, length + 2, BF16)
    w.random(1, [0] * (G * B), [length] * (G * B))
    spare = torch.arange(G * B).int()
    cache = native.PagedCache(ctx, kind, kv_heads=KV, head_dim=D, page_tokens=page, pages=w.cache.c.pages + G * B)
    cache.pool[:w.cache.pool.numel()] = w.cache.pool  # the same pages, and spare ones behind them
    w.cache = cache
    spare = (spare + (cache.c.pages - G * B)).to(DEV)
    parents = [2, 1, 2, 0, 3, 3, 3, -1]  # the last: no beam, itself
    new, spare_out = torch.full_like(w.table, -9), torch.full_like(spare, -9)
    before = w.table.clone()
    cache.reorder(w.table, ints(parents), ints([length] * G), spare, new, spare_out, beams=B)
    assert torch.equal(before, w.table)
    source = [g * B + (p if p >= 0 else b) for g in range(G) for b, p in enumerate(parents[g * B:(g + 1) * B])]
    k, v = w.read([0] * 8, [length] * 8, max(length, 1))
    w.table = new
    kk, vv = w.read([0] * 8, [length] * 8, max(length, 1))
    for r, s in enumerate(source):
        assert torch.equal(kk[r], k[s]) and torch.equal(vv[r], v[s]), r
    full, used = divmod(length, page)
    for r, s in enumerate(source):
        moved = used and r != s
        assert new[r, :full].tolist() == before[s, :full].tolist()
        if full < new.shape[1]:
            assert int(new[r, full]) == int(spare[r] if moved else before[r, full])
        assert new[r, full + 1:].tolist() == before[r, full + 1:].tolist()
        assert int(spare_out[r]) == int(before[r, full] if moved else spare[r])


def test_decoding_with_beams(ctx):
    """Prompt, then steps of append, attention, selection and reorder, two layers with a pool each and one table: at each
    step the rows' attention is that of a cache filled anew with their own histories."""
    torch.manual_seed(0)
    G, B, KV, H, D, page, V, prompt, steps = 2, 3, 2, 4, 64, 16, 300, 13, 9
    S, each = G * B, 2 * ((prompt + steps) // page + 1)
    layers = [native.PagedCache(ctx, "bf16", kv_heads=KV, head_dim=D, page_tokens=page, pages=S * each + S) for _ in range(2)]
    ids = torch.randperm(S * each + S).int().to(DEV)
    table, spare = ids[:S * each].view(S, each).contiguous(), ids[S * each:].contiguous()
    rot = native.Rotary(ctx, prompt + steps, D)
    vocab = torch.randn(V, KV, D, device=DEV), torch.randn(V, KV, D, device=DEV)  # a token's keys and values
    head = torch.randn(H * D, V, device=DEV)
    history = [torch.randint(0, V, (prompt,)).tolist() for _ in range(G) for _ in range(B)]
    for g in range(G):
        for b in range(B):
            history[g * B + b] = list(history[g * B])
    scores = torch.full((G, B), -math.inf, device=DEV)
    scores[:, 0] = 0.0
    ended = torch.zeros(G, B, dtype=torch.int32, device=DEV)
    t = torch.tensor(history, device=DEV)
    for layer, pool in enumerate(layers):
        pool.tokens(table, vocab[0][t], vocab[1][t] + layer, rotary=rot).append(vocab[0][t], vocab[1][t] + layer)
    n = prompt
    for step in range(steps):
        q = torch.randn(S, 1, H, D, device=DEV)
        out = torch.empty(2, S, 1, H, D, device=DEV)
        for layer, pool in enumerate(layers):
            p = pool.queries(table, q, out[layer], most_keys=n, key_lengths=ints([n] * S), query_start=ints([n - 1] * S), rotary=rot,
                             scale=D ** -0.5)
            p.forward(q, out[layer], workspace=buffer(p.workspace_bytes()))
            for r in range(S):
                h = history[r]
                k = R.turn32(vocab[0][h].float().cpu(), rot.table.cpu(), 0, False).bfloat16().float()
                v = (vocab[1][h] + layer).cpu().bfloat16().float()
                val, tol = R.attention("bf16", q[r].cpu(), k, v, scale=D ** -0.5,
                                       turn=lambda x: R.rotary(x[None], [n - 1], D, False)[0][0])
                R.assert_within(out[layer, r], val, tol, f"step {step}, layer {layer}, row {r}")
        logits = (out[0].flatten(1) @ head / 16).view(G, B, V)
        search = native.BeamSearch(ctx, logits, end_token=0)
        tokens, parents, done = (torch.empty(G, B, dtype=torch.int32, device=DEV) for _ in range(3))
        new = torch.empty(G, B, device=DEV)
        search.select(logits, scores, tokens, parents, new, ended=ended, new_ended=done, workspace=buffer(search.workspace_bytes()))
        scores, ended = new, done
        table_out, spare_out = torch.empty_like(table), torch.empty_like(spare)
        for pool in layers:
            pool.reorder(table, parents.view(-1), ints([n] * G), spare, table_out, spare_out, beams=B)
        table, spare = table_out, spare_out
        history = [history[r // B * B + int(p)] + [int(c)] for r, (p, c) in enumerate(zip(parents.view(-1), tokens.view(-1)))]
        last = tokens.view(S, 1).long()
        for layer, pool in enumerate(layers):
            k, v = vocab[0][last], vocab[1][last] + layer
            pool.tokens(table, k, v, start=ints([n] * S), rotary=rot).append(k, v)
        n += 1
        assert len(set(table[:, n // page if n % page else n // page - 1].tolist())) == S  # last pages are rows' own


# ---------------------------------------------------------------- captured, and on other streams

def test_a_step_captured(ctx):
    """Append, attention, selection and reorder in one graph, replayed with other lengths, tokens and tables, eager work
    between; two such graphs with workspaces of their own."""
    S, KV, H, D, page, V = 4, 2, 8, 64, 16, 5000
    w = World(ctx, "int8", S, KV, D, page, 1200, BF16, 64)
    w.random(1, [0] * S, [1000, 17, 500, 0])
    pool0 = w.cache.pool.clone()

    def step():
        st = {n: torch.zeros(S, 1, h, D, dtype=BF16, device=DEV) for n, h in (("k", KV), ("v", KV), ("q", H), ("out", H))}
        st.update(start=ints([0] * S), n=ints([1] * S), logits=torch.zeros(2, 2, V, device=DEV), scores=torch.zeros(2, 2, device=DEV),
                  tokens=ints([[0] * 2] * 2), parents=ints([[0] * 2] * 2), new=torch.zeros(2, 2, device=DEV), table=w.table.clone(),
                  spare=ints([w.cache.c.pages - 1 - i for i in range(3)] + [w.cache.c.pages - 1]), spare_out=ints([0] * S),
                  table_out=torch.zeros_like(w.table), lengths=ints([0, 0]))
        st["a"] = w.cache.tokens(st["table"], st["k"], st["v"], start=st["start"], rotary=w.rotary)
        st["p"] = w.cache.queries(st["table"], st["q"], st["out"], most_keys=1200, key_lengths=st["n"], query_start=st["start"],
                                  rotary=w.rotary)
        st["b"] = native.BeamSearch(ctx, st["logits"])
        st["ws"], st["bs"] = buffer(st["p"].workspace_bytes()), buffer(st["b"].workspace_bytes())
        return st

    def run(st):
        st["a"].append(st["k"], st["v"])
        st["p"].forward(st["q"], st["out"], workspace=st["ws"])
        st["b"].select(st["logits"], st["scores"], st["tokens"], st["parents"], st["new"], workspace=st["bs"])
        w.cache.reorder(st["table"], st["parents"].view(-1), st["lengths"], st["spare"], st["table_out"], st["spare_out"], beams=2)

    stream = torch.cuda.Stream()
    states, graphs = [step(), step()], []
    for st in states:
        with torch.cuda.stream(stream):
            ctx.set_stream(stream.cuda_stream)
            run(st)
        stream.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            run(st)
        graphs.append(g)
    ctx.set_stream(0)
    eager = step()
    names = ("out", "tokens", "parents", "new", "table_out", "spare_out")
    for i in range(4):
        for st in (*states, eager):
            for n, x in (("k", 1), ("v", 2), ("q", 3)):
                st[n].copy_(randn(100 * i + x, *st[n].shape, dtype=BF16))
            st["start"].copy_(ints([1000 + i, 17, 500 + 16 * i, i]))
            st["n"].copy_(st["start"] + 1)
            st["logits"].copy_(randn(100 * i + 4, 2, 2, V))
            st["scores"].copy_(randn(100 * i + 5, 2, 2))
            st["lengths"].copy_(ints([16 * i, 32]))
        results = []
        for what in (lambda: run(eager), graphs[0].replay, graphs[1].replay):
            w.cache.pool.copy_(pool0)
            torch.cuda.synchronize()
            what()
            torch.cuda.synchronize()
            results.append(w.cache.pool.clone())
        assert torch.equal(results[0], results[1]) and torch.equal(results[0], results[2])
        for st in states:  # bits: sequence 2 leaves out tokens, whose block's scale is what the pool began with, a NaN
            assert [n for n in names if not torch.equal(st[n].view(torch.uint8), eager[n].view(torch.uint8))] == [], i
            assert bool(st["out"][[0, 1, 3]].isfinite().all())
        pool0.copy_(results[0])


def test_other_stream(ctx):
    w = World(ctx, "bf16", 2, 1, 64, 16, 100, F32, 64)
    w.random(1, [0, 0], [90, 33])
    q = randn(2, 2, 1, 2, 64)
    want = attend(w, q, start=[89, 32], scale=0.125)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    with torch.cuda.stream(stream):
        got = attend(w, q, start=[89, 32], scale=0.125)
        stream.synchronize()
    ctx.set_stream(0)
    assert torch.equal(got, want)

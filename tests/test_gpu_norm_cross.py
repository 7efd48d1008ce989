"""Layer norm, cross attention and the relative position bias on the GPU, forward and backward, against their
definitions in 64 bits (norm_cross_ref.py), at the sizes, masks, strides and values where they can go wrong."""

import math

import pytest
import torch

import norm_cross_ref as R
from helpers import gpu_available

pytestmark = pytest.mark.gpu

if gpu_available():
    from vocalarc_hip import native

DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
NAN = math.nan


@pytest.fixture(scope="module")
def ctx():
    c = native.Context()
    yield c
    c.close()


def randn(seed, *shape, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g).to(dtype)


def buf(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=DEV)


# --------------------------------------------------------------- layer norm

def norm(ctx, x, gamma, beta, dy=None, eps=1e-5, pitch=None, weights=True):
    """y (and dx, dgamma, dbeta) of x [rows][dim]; pitch: rows that far apart, with NaN between them."""
    rows, dim = x.shape
    bf16 = x.dtype == BF16

    def spread(t):
        if pitch is None:
            return t.contiguous(), dim
        wide = torch.full((rows, pitch), NAN, dtype=t.dtype, device=DEV)
        wide[:, :dim] = t
        return wide, pitch
    xs, ld = spread(x)
    y, _ = spread(torch.full_like(x, NAN))
    stats = torch.empty(rows, 2, device=DEV)
    ctx.layernorm(xs, gamma, beta, y, rows, dim, eps=eps, stats=stats, ldx=ld, ldy=ld, bf16=bf16)
    r = {"y": y[:, :dim]}
    if dy is not None:
        dys, _ = spread(dy)
        dx, _ = spread(torch.full_like(x, NAN))
        dgamma, dbeta = (torch.full((dim,), NAN, device=DEV) for _ in range(2)) if weights else (None, None)
        ws = buf(ctx.layernorm_workspace_bytes(rows, dim)) if weights else None
        ctx.layernorm_backward(dys, xs, gamma, stats, dx, rows, dim, dgamma=dgamma, dbeta=dbeta, workspace=ws,
                               lddy=ld, ldx=ld, lddx=ld, bf16=bf16)
        r["dx"] = dx[:, :dim]
        if weights:
            r.update(dgamma=dgamma, dbeta=dbeta)
        if pitch:
            assert bool(dx[:, dim:].isnan().all())
    if pitch:
        assert bool(y[:, dim:].isnan().all())
    return r


def check_norm(ctx, x, gamma, beta, dy, what, **kw):
    got = norm(ctx, x, gamma, beta, dy, **kw)
    val, tol = R.layernorm(x, gamma, beta, kw.get("eps", 1e-5), dy)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{what} {n}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 1), (1, 384), (5, 3), (7, 63), (4, 64), (9, 65), (33, 256), (2, 257),
                                      (801, 384), (6, 512), (5, 513), (2, 1023), (3, 1024), (2, 1025), (4, 2048),
                                      (3, 2052), (2, 4096), (2, 4097), (3, 8192), (2, 16383), (2, 16384)])
def test_layernorm(ctx, rows, dim, dtype):
    x = randn(1, rows, dim) * 2 + 0.5
    check_norm(ctx, x.to(dtype), 1 + 0.1 * randn(2, dim), randn(3, dim), randn(4, rows, dim, dtype=dtype),
               f"{rows}x{dim}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,dim", [(2049, 384), (5000, 65), (10007, 20), (700, 2048), (1500, 1025)])
def test_layernorm_many_rows(ctx, rows, dim, dtype):
    """More rows than the backward pass has workgroups."""
    check_norm(ctx, randn(1, rows, dim, dtype=dtype), 1 + 0.1 * randn(2, dim), None, randn(4, rows, dim, dtype=dtype),
               f"{rows}x{dim}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [1, 7, 20, 72, 130, 200, 300, 384, 500, 512, 513, 700, 1023, 1024, 1500, 2047])
def test_layernorm_more_rows(ctx, dim, dtype):
    """Enough rows for several to a wave, at each number of a row's lanes and of a lane's elements."""
    check_norm(ctx, randn(1, 4160, dim, dtype=dtype), 1 + 0.1 * randn(2, dim), randn(3, dim),
               randn(4, 4160, dim, dtype=dtype), f"4160x{dim}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dim,pitch", [(384, 400), (384, 385), (65, 128), (1028, 1030), (5000, 5004)])
def test_layernorm_pitch(ctx, dim, pitch, dtype):
    """Rows with gaps between them, which are neither read nor written."""
    check_norm(ctx, randn(1, 11, dim, dtype=dtype), 1 + 0.1 * randn(2, dim), randn(3, dim),
               randn(4, 11, dim, dtype=dtype), f"{dim} of {pitch}", pitch=pitch)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layernorm_unaligned(ctx, dtype):
    """Tensors and weights that begin one element past a vector."""
    rows, dim = 9, 384
    x, dy = randn(1, rows * dim + 1, dtype=dtype)[1:].view(rows, dim), randn(2, rows * dim + 1, dtype=dtype)[1:].view(rows, dim)
    gamma, beta = 1 + 0.1 * randn(3, dim + 1)[1:], randn(4, dim + 1)[1:]
    check_norm(ctx, x, gamma, beta, dy, "unaligned")


def test_layernorm_beyond_one_launch(ctx):
    """More rows than one launch has places for, at single-column pitch: (a, b) has the norm (+-1, -+1) where a != b."""
    rows = (1 << 28) + 5
    x = torch.zeros(rows, 2, dtype=BF16, device=DEV)
    x[:, 0] = 1
    x[-7:] = torch.tensor([0, 1], dtype=BF16, device=DEV)
    gamma = torch.tensor([2.0, 4.0], device=DEV)
    st = torch.full((rows, 2), NAN, device=DEV)
    ctx.layernorm(x, gamma, None, x, rows, 2, eps=0.0, stats=st, bf16=True)
    want = torch.tensor([2.0, -4.0], dtype=BF16, device=DEV)
    assert bool((x[:-7] == want).all()) and bool((x[-7:] == -want).all())
    assert bool((st == torch.tensor([0.5, 2.0], device=DEV)).all())


def test_layernorm_values(ctx):
    """Rows far from 0 (the variance is taken about the mean), constant rows (variance 0, only eps), eps 0, tiny and
    huge rows; no weights' gradients wanted."""
    dim = 384
    gamma, beta = 1 + 0.1 * randn(2, dim), randn(3, dim)
    x = randn(1, 6, dim)
    x[0] += 1000
    x[1] = 7.25
    x[2] *= 1e-12
    x[3] *= 1e15
    check_norm(ctx, x, gamma, beta, randn(4, 6, dim), "values")
    check_norm(ctx, x[3:], gamma, beta, randn(4, 3, dim), "eps 0", eps=0.0, weights=False)
    bad = x.clone()
    bad[4, 17] = math.inf
    bad[5, 3] = NAN
    y = norm(ctx, bad, gamma, beta)["y"]
    assert bool(y[4:].isnan().any(1).all()) and bool(y[:4].isfinite().all())


def test_layernorm_in_place_and_repeat(ctx):
    """y on x, dx on dy and dx on x; equal calls give equal bits."""
    rows, dim = 1203, 384
    for dtype in (F32, BF16):
        x, dy, gamma = randn(1, rows, dim, dtype=dtype), randn(2, rows, dim, dtype=dtype), 1 + 0.1 * randn(3, dim)
        a, b = norm(ctx, x, gamma, None, dy), norm(ctx, x, gamma, None, dy)
        assert all(torch.equal(a[n], b[n]) for n in a)
        bf16 = dtype == BF16
        stats, ws = torch.empty(rows, 2, device=DEV), buf(ctx.layernorm_workspace_bytes(rows, dim))
        y = x.clone()
        ctx.layernorm(y, gamma, None, y, rows, dim, stats=stats, bf16=bf16)
        assert torch.equal(y, a["y"])
        for place in ("dy", "x"):
            t = {"dy": dy.clone(), "x": x.clone()}
            dg, db = torch.empty(dim, device=DEV), torch.empty(dim, device=DEV)
            ctx.layernorm_backward(t["dy"], t["x"], gamma, stats, t[place], rows, dim, dgamma=dg, dbeta=db,
                                   workspace=ws, bf16=bf16)
            assert torch.equal(t[place], a["dx"]) and torch.equal(dg, a["dgamma"]) and torch.equal(db, a["dbeta"])


def test_layernorm_no_rows_and_refusals(ctx):
    gamma = torch.ones(8, device=DEV)
    dg, db = torch.full((8,), NAN, device=DEV), torch.full((8,), NAN, device=DEV)
    e = torch.empty(0, 8, device=DEV)
    ctx.layernorm(e, gamma, None, e, 0, 8)
    ctx.layernorm_backward(e, e, gamma, e, e, 0, 8, dgamma=dg, dbeta=db, workspace=buf(64))
    assert not bool(dg.any()) and not bool(db.any())
    x, st = torch.ones(2, 8, device=DEV), torch.empty(2, 2, device=DEV)
    for bad in (dict(rows=-1), dict(dim=0), dict(dim=16385), dict(ldx=7), dict(ldy=4), dict(eps=NAN), dict(eps=-1.0),
                dict(eps=math.inf)):
        with pytest.raises(native.NativeError, match="vh_layernorm"):
            ctx.layernorm(x, gamma, None, x, **{**dict(rows=2, dim=8), **bad})
    with pytest.raises(native.NativeError, match="workspace"):
        ctx.layernorm_backward(x, x, gamma, st, x, 2, 8, dgamma=dg)
    with pytest.raises(native.NativeError, match="workspace"):
        ctx.layernorm_backward(x, x, gamma, st, x, 2, 8, dgamma=dg, workspace=buf(256)[4:])
    assert bool((x == 1).all())


def test_layernorm_gradient_by_differences(ctx):
    """dx, dgamma and dbeta against central differences of the forward pass in a random direction: of third order in
    the step, and the forward's own roundings over it."""
    rows, dim = 5, 64
    x, dy, gamma, beta = randn(1, rows, dim), randn(2, rows, dim), 1 + 0.1 * randn(3, dim), randn(4, dim)
    r = norm(ctx, x, gamma, beta, dy)
    step = 2.0 ** -7
    f = lambda x, g, b: float((norm(ctx, x, g, b)["y"].double() * dy.double()).sum())  # noqa: E731
    for name, i in (("dx", 0), ("dgamma", 1), ("dbeta", 2)):
        args = [x, gamma, beta]
        d = randn(5 + i, *args[i].shape)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * step * d
            ends.append(f(*moved))
        diff, want = (ends[0] - ends[1]) / (2 * step), float((r[name].double() * d.double()).sum())
        # y's roundings (and the moved input's), 8 half steps of |y| <= 8 in each of rows * dim terms, added at random
        noise = 8 * 8 * R.U * math.sqrt(rows * dim) * 4 / step
        assert abs(diff - want) <= noise + 40 * step ** 2 * rows * dim ** 0.5, name


# ---------------------------------------------------------------- attention

def views(kind, t):
    """t [S][L][H][64] on other strides: heads before rows, rows outermost, a slice of something wider."""
    S, L, H, D = t.shape
    if kind == "bhld":
        return t.transpose(1, 2).contiguous().transpose(1, 2)
    if kind == "lbhd":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    if kind == "slice":
        wide = torch.full((S, L, H + 1, 2 * D), NAN, dtype=t.dtype, device=DEV)
        wide[:, :, :H, D:] = t
        return wide[:, :, :H, D:]
    return t.contiguous()


def empty_as(t):
    """NaN on t's strides."""
    e = torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=DEV) if t.numel() else t.clone()
    return e.fill_(NAN)


def ints(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device=DEV)


def attend(ctx, q, k, v, dout=None, dkv=True, **kw):
    for n in ("query_lengths", "key_lengths", "query_start"):
        kw[n] = ints(kw.get(n))
    out = empty_as(q)
    p = native.CrossAttention(ctx, q, k, v, out, **kw)
    ws = buf(max(p.workspace_bytes(False), p.workspace_bytes(True) if dout is not None else 0)).fill_(0xff)
    saved = buf(p.saved_bytes()).fill_(0xff) if dout is not None else None
    p.forward(q, k, v, out, saved=saved, workspace=ws)
    r = {"out": out}
    if dout is not None:
        r["dq"] = empty_as(q)
        r["dk"], r["dv"] = (empty_as(k), empty_as(v)) if dkv else (None, None)
        r["dbias"] = torch.full_like(kw["bias_table"], NAN) if kw.get("bias_table") is not None else None
        ws.fill_(0xff)
        dout = dout.as_strided(dout.shape, dout.stride()) if dout.stride() == out.stride() else \
            empty_as(out).copy_(dout)
        p.backward(q, k, v, out, saved, dout, r["dq"], r["dk"], r["dv"], dbias=r["dbias"], workspace=ws)
    return {n: t for n, t in r.items() if t is not None}


def make(S, H, KV, Lq, Lk, dtype, seed=0, size=1.0, strides=("", "", "")):
    q, k, v, dout = (randn(4 * seed + i, S, L, h, 64) for i, (L, h) in
                     enumerate(((Lq, H), (Lk, KV), (Lk, KV), (Lq, H))))
    q, k, v, dout = (q * size).to(dtype), k.to(dtype), v.to(dtype), dout.to(dtype)
    return views(strides[0], q), views(strides[1], k), views(strides[2], v), dout


def check(ctx, q, k, v, dout, what, **kw):
    got = attend(ctx, q, k, v, dout, **kw)
    val, tol = R.attention(q, k, v, dout=dout, **kw)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{what} {n}")
    # without state for the backward pass (bf16: probabilities in one piece)
    R.assert_within(attend(ctx, q, k, v, **kw)["out"], val["out"], tol["out"], f"{what} out alone")
    return got


SIZES = [(1, 1, 1, 1, 1), (1, 8, 8, 1, 77), (2, 4, 4, 31, 33), (1, 2, 2, 32, 32), (2, 2, 1, 33, 31), (1, 4, 2, 128, 64),
         (3, 6, 2, 129, 65), (1, 1, 1, 5, 1000), (1, 2, 2, 257, 3), (2, 8, 2, 3, 500), (1, 3, 3, 401, 389),
         (1, 16, 2, 2, 70), (5, 4, 1, 1, 300), (1, 1, 1, 1, 4097), (2, 32, 8, 1, 640)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_cross(ctx, size, dtype):
    q, k, v, dout = make(*size, dtype)
    check(ctx, q, k, v, dout, str(size))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(3, 4, 2, 70, 90), (4, 2, 2, 1, 400), (3, 8, 4, 3, 129), (2, 2, 1, 140, 33)], ids=str)
def test_lengths(ctx, size, dtype):
    """Ragged lengths, empty sequences on both sides, lengths beyond the tensors' and below 0; what lies behind the
    lengths is NaN and infinity, and their rows are zeros."""
    S, H, KV, Lq, Lk = size
    qlens, klens = [Lq - Lq // 3, Lq + 5, Lq // 2, 0][:S], [Lk // 2, Lk, 0, 7][:S]
    if S == 2:
        klens = [-3, Lk + 9]
    q, k, v, dout = make(*size, dtype)
    for s in range(S):
        q[s, max(qlens[s], 0):], dout[s, max(qlens[s], 0):] = NAN, math.inf
        k[s, max(klens[s], 0):], v[s, max(klens[s], 0):] = math.inf, NAN
    got = check(ctx, q, k, v, dout, str(size), query_lengths=qlens, key_lengths=klens)
    for s in range(S):
        assert not bool(got["out"][s, max(qlens[s], 0):].any()) and not bool(got["dk"][s, max(klens[s], 0):].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size,start", [((2, 4, 4, 70, 70), None), ((3, 4, 2, 1, 300), [299, 0, 150]),
                                        ((3, 2, 2, 5, 200), [195, 0, 77]), ((2, 2, 1, 40, 130), [90, 30]),
                                        ((2, 2, 2, 150, 60), [0, -40]), ((3, 2, 2, 33, 64), [-1000, 2 ** 31 - 1, 1000]),
                                        ((1, 4, 1, 130, 400), [-2 ** 31])], ids=str)
def test_causal(ctx, size, start, dtype):
    """A row that lies before every key sees none."""
    q, k, v, dout = make(*size, dtype)
    lens = [size[4] - 3 * s for s in range(size[0])]
    check(ctx, q, k, v, dout, str(size), causal=True, query_start=start, key_lengths=lens)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets", [0, 32])
@pytest.mark.parametrize("size,start", [((2, 8, 2, 1, 300), [100, 17]), ((2, 4, 4, 5, 90), [60, 0]),
                                        ((2, 4, 2, 70, 400), [200, 3]), ((5, 16, 16, 600, 700), [40, 0, -20, 77, 99])],
                         ids=str)
def test_causal_cache_not_yet_filled(ctx, size, start, buckets, dtype):
    """Keys that come after every query hold NaN and infinity, as memory that a cache has not written: nobody sees
    them."""
    S, H, KV, Lq, Lk = size
    q, k, v, dout = make(*size, dtype)
    kw = dict(causal=True, query_start=start)
    if buckets:
        kw.update(bias_table=randn(9, buckets, H), bidirectional=False)
    val, tol = R.attention(q, k, v, dout=dout, **kw)
    for s in range(S):
        end = start[s] + Lq
        k[s, end::2], k[s, end + 1::2], v[s, end::2], v[s, end + 1::2] = NAN, math.inf, -math.inf, NAN
    got = attend(ctx, q, k, v, dout, **kw)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{size} {n}")
    R.assert_within(attend(ctx, q, k, v, **kw)["out"], val["out"], tol["out"], f"{size} out alone")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size,buckets,max_distance,bidirectional,start", [
    ((1, 2, 2, 1, 1), 32, 128, True, None), ((2, 4, 4, 70, 70), 32, 128, True, None),
    ((2, 4, 2, 300, 170), 32, 128, False, None), ((1, 2, 1, 170, 430), 32, 128, True, None),
    ((2, 8, 2, 1, 500), 32, 128, False, [499, 200]), ((2, 4, 4, 3, 333), 16, 96, True, [330, -20]),
    ((1, 2, 2, 200, 200), 128, 4096, True, None), ((1, 2, 2, 200, 200), 4, 2, True, None),
    ((1, 2, 2, 150, 300), 2, 3, False, [60]), ((2, 2, 2, 40, 600), 64, 300, True, [900, 280])], ids=str)
def test_bias(ctx, size, buckets, max_distance, bidirectional, start, causal, dtype):
    q, k, v, dout = make(*size, dtype)
    check(ctx, q, k, v, dout, str(size), causal=causal, query_start=start, bias_table=randn(9, buckets, size[1]),
          max_distance=max_distance, bidirectional=bidirectional, scale=0.1)


# many rows, sequences and heads: workgroups of 128 rows (forward: of 64 below 1024 of them), dk and dv of all heads
# that share their keys in one workgroup or each head's on its own
MANY = [(13, 16, 16, 600, 97), (5, 16, 16, 600, 600), (10, 16, 8, 300, 600), (32, 12, 12, 64, 70), (8, 16, 8, 200, 130),
        (6, 16, 2, 260, 300), (70, 16, 16, 40, 33)]


def few(bound, n):
    return [int(bound * (i % n) / (n - 1)) for i in range(n)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", MANY, ids=str)
def test_many(ctx, size, dtype):
    q, k, v, dout = make(*size, dtype)
    check(ctx, q, k, v, dout, str(size))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal,buckets", [(True, 0), (False, 32), (True, 32)])
@pytest.mark.parametrize("size", MANY, ids=str)
def test_many_ragged(ctx, size, causal, buckets, dtype):
    """Lengths from none to all, NaN behind them; equal calls give equal bits."""
    S, H, KV, Lq, Lk = size
    qlens, klens = few(Lq, S), few(Lk, S)[::-1]
    klens[S // 2] = Lk
    q, k, v, dout = make(*size, dtype)
    for s in range(S):
        q[s, qlens[s]:], dout[s, qlens[s]:], k[s, klens[s]:], v[s, klens[s]:] = NAN, math.inf, math.inf, NAN
    kw = dict(causal=causal, query_lengths=qlens, key_lengths=klens, query_start=[Lk - Lq + 40 * (s % 3 - 1) for s in range(S)])
    if buckets:
        kw.update(bias_table=randn(9, buckets, H), max_distance=128, bidirectional=not causal)
    got = check(ctx, q, k, v, dout, str(size), **kw)
    again = attend(ctx, q, k, v, dout, **kw)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("size,start", [((2, 8, 2, 1, 5000), [4999, 1300]), ((1, 4, 1, 9, 4100), [4000]),
                                        ((2, 4, 2, 40, 2500), [2460, -7]), ((1, 2, 2, 1300, 64), [0]),
                                        ((1, 4, 2, 100, 100), [2 ** 31 - 1]), ((1, 4, 2, 100, 100), [-2 ** 31])], ids=str)
def test_bias_in_pieces(ctx, size, start, causal, dtype):
    """Few rows over many keys, and few keys under many rows, whose sums are joined; starts out of reach."""
    q, k, v, dout = make(*size, dtype)
    check(ctx, q, k, v, dout, str(size), causal=causal, query_start=start, bias_table=randn(9, 32, size[1]),
          key_lengths=[size[4] - 30 * s for s in range(size[0])])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_bias_that_hides(ctx, dtype):
    """Buckets at -inf hide their pairs, some rows' all of them (0, and no gradient); buckets at the type's lowest value
    leave a row of them alone uniform, as sums in fp32 do, and hide the pair beside others."""
    q, k, v, dout = make(1, 2, 2, 200, 20, dtype, size=0.1)
    table = randn(9, 32, 2)
    table[15] = -math.inf  # the past from the last border on
    got = check(ctx, q, k, v, dout, "-inf", bias_table=table)
    assert not bool(got["out"][0, 150:].any()) and not bool(got["dq"][0, 150:].any())
    table[15] = torch.finfo(F32).min
    got = attend(ctx, q, k, v, dout, bias_table=table)
    alone = got["out"][0, 150:].double()
    mean = v.double().mean(1).expand(50, 2, 64)
    # 20 equal probabilities: each off by 2 U (bf16: and its rounding), 20 sums, the rounding of the result
    half = R.HALF[dtype]
    bound = (half + 24 * R.U) * v.double().abs().mean(1) + (half + R.U) * mean.abs()
    R.assert_within(alone, mean, bound, "lowest")
    assert all(bool(t.isfinite().all()) for t in got.values())
    # beside visible pairs both hide alike
    hidden = table.clone()
    hidden[15] = -math.inf
    a, b = (attend(ctx, q, k, v, bias_table=t)["out"][0, :100] for t in (table, hidden))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("causal", [False, True])
def test_bias_that_hides_many(ctx, causal, dtype):
    """The same in workgroups of 128 rows; scores of hundreds there."""
    q, k, v, dout = make(8, 16, 16, 400, 33, dtype, size=20.0)
    table = randn(9, 32, 16)
    table[15] = -math.inf
    got = check(ctx, q, k, v, dout, "-inf", bias_table=table, causal=causal)
    assert not bool(got["out"][:, 170:].any()) and not bool(got["dq"][:, 170:].any())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("strides", [("bhld", "bhld", "bhld"), ("lbhd", "slice", ""), ("slice", "lbhd", "bhld"),
                                     ("", "slice", "lbhd")], ids=str)
def test_strides(ctx, strides, dtype):
    q, k, v, dout = make(2, 4, 2, 70, 45, dtype, strides=strides)
    check(ctx, q, k, v, dout, str(strides), bias_table=randn(9, 32, 4), key_lengths=[45, 20])
    q1, k1, v1, dout1 = make(2, 4, 2, 1, 300, dtype, strides=strides)
    check(ctx, q1, k1, v1, dout1, str(strides), key_lengths=[300, 20])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_single_ones(ctx, dtype):
    """One row, one head, one sequence: whatever their strides are."""
    for size in ((1, 1, 1, 1, 40), (1, 2, 2, 1, 1), (3, 1, 1, 1, 1), (1, 1, 1, 50, 40)):
        q, k, v, dout = make(*size, dtype)
        odd = lambda t: t.as_strided(t.shape, [n if m > 1 else 77 for m, n in zip(t.shape[:3], t.stride())] + [1])  # noqa: E731
        check(ctx, odd(q), odd(k), odd(v), dout, str(size))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shared_inputs(ctx, dtype):
    """One sequence's keys read by every sequence, one head's by all (strides of 0): forward only."""
    q, k, v, _ = make(3, 4, 4, 40, 50, dtype)
    k, v = k[:1].expand(3, -1, -1, -1), v[:, :, :1].expand(-1, -1, 4, -1)
    val, tol = R.attention(q, k, v)
    R.assert_within(attend(ctx, q, k, v)["out"], val["out"], tol["out"], "shared")
    out = torch.empty_like(q)
    p = native.CrossAttention(ctx, q, k, v, out)
    with pytest.raises(native.NativeError, match="overlap"):
        p.workspace_bytes(True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [30.0, 1e-3, 200.0])
def test_peaked_and_flat(ctx, size, dtype):
    """Scores of hundreds, where one key takes all, and of nearly nothing."""
    q, k, v, dout = make(2, 2, 2, 65, 333, dtype, size=size)
    check(ctx, q, k, v, dout, str(size))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.0])
def test_scale(ctx, scale, dtype):
    q, k, v, dout = make(2, 4, 2, 45, 75, dtype)
    check(ctx, q, k, v, dout, str(scale), scale=scale, causal=True, query_start=[20, 0])
    check(ctx, q, k, v, dout, str(scale), scale=scale, bias_table=randn(9, 32, 4))


def test_values_past_range(ctx):
    """NaN and infinity in a query stay in its row, in a key or value go where it is seen."""
    q, k, v, _ = make(1, 2, 2, 70, 60, F32)
    q[0, 3, 0, 5], q[0, 4, 1, 7] = NAN, math.inf
    out = attend(ctx, q, k, v)["out"]
    bad = out.isnan().any(-1)[0]
    assert bad.nonzero().tolist() == [[3, 0], [4, 1]]
    q, k, v, _ = make(1, 1, 1, 70, 70, BF16)
    k[0, 40, 0, 0] = NAN
    out = attend(ctx, q, k, v, causal=True)["out"][0, :, 0]
    assert bool(out[40:].isnan().any(-1).all()) and bool(out[:32].isfinite().all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_keys_no_rows(ctx, dtype):
    for S, Lq, Lk in ((2, 5, 0), (2, 0, 5), (0, 5, 5), (0, 0, 0)):
        q, k, v, dout = make(S, 2, 2, Lq, Lk, dtype)
        r = attend(ctx, q, k, v, dout, bias_table=randn(9, 32, 2))
        assert not any(bool(t.any()) for t in r.values()), (S, Lq, Lk)
        assert not bool(r["dbias"].isnan().any())


def test_frozen_states(ctx):
    """dk and dv not wanted: dq and the table's gradient are the same."""
    q, k, v, dout = make(2, 4, 2, 70, 45, BF16)
    table = randn(9, 32, 4)
    a, b = attend(ctx, q, k, v, dout, bias_table=table), attend(ctx, q, k, v, dout, dkv=False, bias_table=table)
    assert torch.equal(a["dq"], b["dq"]) and torch.equal(a["dbias"], b["dbias"]) and "dk" not in b


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits(ctx, dtype):
    for size in ((2, 4, 2, 300, 290), (4, 8, 2, 1, 3000)):
        q, k, v, dout = make(*size, dtype)
        kw = dict(bias_table=randn(9, 32, size[1]), key_lengths=[size[4] - 5 * i for i in range(size[0])])
        a, b = attend(ctx, q, k, v, dout, **kw), attend(ctx, q, k, v, dout, **kw)
        assert all(torch.equal(a[n], b[n]) for n in a)


def test_long_cache(ctx):
    """Keys beyond 2^32 bytes from their first: rows 8 MiB apart and the same few rows read at the end."""
    L, row = 600, (1 << 23) // 4
    store = torch.empty(L * row, device=DEV)
    kv = store.as_strided((1, L, 2, 64), (0, row, 64, 1))
    kv.copy_(randn(1, 1, L, 2, 64))
    q, v = randn(2, 1, 3, 2, 64), randn(3, 1, L, 2, 64)
    val, tol = R.attention(q, kv, v)
    R.assert_within(attend(ctx, q, kv, v)["out"], val["out"], tol["out"], "k")
    val, tol = R.attention(q, v, kv)
    R.assert_within(attend(ctx, q, v, kv)["out"], val["out"], tol["out"], "v")


def test_refusals(ctx):
    q, k, v, dout = make(1, 2, 2, 3, 5, F32)
    out = torch.full_like(q, 5.0)
    p = native.CrossAttention(ctx, q, k, v, out)
    ws, saved = buf(p.workspace_bytes(True)), buf(p.saved_bytes())
    off = torch.empty(q.numel() + 1, device=DEV)[1:].view(q.shape)
    with pytest.raises(native.NativeError, match="aligned"):
        p.forward(off, k, v, out, workspace=ws)
    with pytest.raises(native.NativeError, match="aligned"):
        p.forward(q, k, v, off, workspace=ws)
    with pytest.raises(native.NativeError, match="together"):
        p.backward(q, k, v, out, saved, dout, torch.empty_like(q), dk=torch.empty_like(k), workspace=ws)
    with pytest.raises(native.NativeError, match="bias table"):
        p.backward(q, k, v, out, saved, dout, torch.empty_like(q), dbias=torch.empty(32, 2, device=DEV), workspace=ws)
    with pytest.raises(native.NativeError, match="workspace"):
        p.backward(q, k, v, out, saved, dout, torch.empty_like(q))
    p.c.heads = 3
    with pytest.raises(native.NativeError, match="heads"):
        p.forward(q, k, v, out, workspace=ws)
    assert bool((out == 5.0).all())


def test_keys_without_rows(ctx):
    """No query rows: dk and dv are 0, and null keys are refused there too."""
    q, k, v, dout = make(2, 2, 2, 0, 5, F32)
    p = native.CrossAttention(ctx, q, k, v, q)
    dk, dv, ws = torch.full_like(k, NAN), torch.full_like(k, NAN), buf(p.workspace_bytes(True))
    null = lambda t: None if not t.numel() else t.data_ptr()  # noqa: E731
    call = lambda k: native.lib().vh_cross_attention_backward(  # noqa: E731
        ctx.h, p._ref, null(q), k, v.data_ptr(), null(q), ws.data_ptr(), null(dout), null(q), dk.data_ptr(),
        dv.data_ptr(), None, ws.data_ptr())
    assert not call(None) and "null" in native.last_error()
    assert call(k.data_ptr())
    torch.cuda.synchronize()
    assert not bool(dk.any()) and not bool(dv.any())


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_by_differences(ctx, causal):
    """dq, dk, dv and dbias against central differences of the forward pass in a random direction."""
    S, H, KV, Lq, Lk = 2, 2, 1, 9, 40
    q, k, v, dout = make(S, H, KV, Lq, Lk, F32)
    table = randn(9, 8, H)
    kw = dict(causal=causal, query_start=[20, 3], key_lengths=[40, 17], max_distance=16)
    r = attend(ctx, q, k, v, dout, bias_table=table, **kw)
    f = lambda q, k, v, t: float((attend(ctx, q, k, v, bias_table=t, **kw)["out"].double() * dout.double()).sum())  # noqa: E731
    step = 2.0 ** -6
    for i, name in enumerate(("dq", "dk", "dv", "dbias")):
        args = [q, k, v, table]
        d = randn(20 + i, *args[i].shape)
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[i] = args[i] + sign * step * d
            ends.append(f(*moved))
        diff, want = (ends[0] - ends[1]) / (2 * step), float((r[name].double() * d.double()).sum())
        # the forward's roundings, 64 half steps of |out| <= 4 in each term, added at random, over the step; and the
        # third derivative: every row's share of it is below 2 |dout| in norm (scores move by about 1 per unit)
        noise = 64 * 4 * R.U * math.sqrt(out_terms := S * H * Lq * 64) / step
        assert abs(diff - want) <= noise + step ** 2 * 2 * math.sqrt(out_terms) * 8, (name, diff, want)


# ------------------------------------------------ together, streams and graphs

def block(ctx, t, step=True):
    """A conditioned decoder's layer as a program runs it: norm, biased attention, residual, norm, cross attention,
    residual, and back."""
    S, L, H, E, dim = t["S"], t["L"], t["H"], t["E"], t["H"] * 64
    ctx.layernorm(t["x"], t["g1"], t["b1"], t["n1"], S * L, dim, stats=t["st1"])
    t["self"].forward(t["n1"], t["n1"], t["n1"], t["a"], saved=t["save1"], workspace=t["ws1"])
    torch.add(t["x"], t["a"].view(S * L, dim), out=t["y"])
    ctx.layernorm(t["y"], t["g2"], t["b2"], t["n2"], S * L, dim, stats=t["st2"])
    t["cross"].forward(t["n2"], t["enc"], t["enc"], t["c"], saved=t["save2"], workspace=t["ws2"])
    torch.add(t["y"], t["c"].view(S * L, dim), out=t["z"])
    # back from dz
    t["cross"].backward(t["n2"], t["enc"], t["enc"], t["c"], t["save2"], t["dz"], t["dn2"], t["dek"], t["dev"],
                        workspace=t["ws2"])
    ctx.layernorm_backward(t["dn2"], t["y"], t["g2"], t["st2"], t["dy"], S * L, dim, dgamma=t["dg2"], dbeta=t["db2"],
                           workspace=t["wsn"])
    torch.add(t["dy"], t["dz"].view(S * L, dim), out=t["dy"])
    t["self"].backward(t["n1"], t["n1"], t["n1"], t["a"], t["save1"], t["dy"], t["dn1"], t["dk1"], t["dv1"],
                       dbias=t["dtable"], workspace=t["ws1"])
    t["dn1"] += t["dk1"]
    t["dn1"] += t["dv1"]
    ctx.layernorm_backward(t["dn1"], t["x"], t["g1"], t["st1"], t["dx"], S * L, dim, dgamma=t["dg1"], dbeta=t["db1"],
                           workspace=t["wsn"])
    torch.add(t["dx"], t["dy"], out=t["dx"])


OUTS = ("z", "dx", "dg1", "db1", "dg2", "db2", "dtable", "dek", "dev")


def block_state(ctx, seed=0, S=2, L=75, H=4, E=33):
    dim = H * 64
    t = {"S": S, "L": L, "H": H, "E": E}
    t["x"] = randn(seed, S * L, dim)
    for i, n in enumerate(("g1", "g2")):
        t[n] = 1 + 0.1 * randn(seed + 10 + i, dim)
    for i, n in enumerate(("b1", "b2")):
        t[n] = 0.1 * randn(seed + 12 + i, dim)
    t["table"], t["enc"] = randn(seed + 14, 32, H), randn(seed + 15, S, E, H, 64)
    t["dz"] = randn(seed + 16, S, L, H, 64)
    for n in ("y", "z", "dy", "dx"):
        t[n] = torch.empty(S * L, dim, device=DEV)
    for n in ("n1", "n2", "a", "c", "dn1", "dn2", "dk1", "dv1"):
        t[n] = torch.empty(S, L, H, 64, device=DEV)
    t["dek"], t["dev"], t["dtable"] = torch.empty_like(t["enc"]), torch.empty_like(t["enc"]), torch.empty_like(t["table"])
    for n in ("dg1", "dg2", "db1", "db2"):
        t[n] = torch.empty(dim, device=DEV)
    t["st1"], t["st2"] = torch.empty(S * L, 2, device=DEV), torch.empty(S * L, 2, device=DEV)
    t["klens"] = ints([E, E - 9] + [E] * (S - 2))
    t["self"] = native.CrossAttention(ctx, t["n1"], t["n1"], t["n1"], t["a"], causal=True, bias_table=t["table"],
                                      bidirectional=False)
    t["cross"] = native.CrossAttention(ctx, t["n2"], t["enc"], t["enc"], t["c"], key_lengths=t["klens"])
    for i, p in ((1, t["self"]), (2, t["cross"])):
        t[f"save{i}"], t[f"ws{i}"] = buf(p.saved_bytes()), buf(max(p.workspace_bytes(False), p.workspace_bytes(True)))
    t["wsn"] = buf(ctx.layernorm_workspace_bytes(S * L, dim))
    return t


def block_reference(t):
    """The block's outputs by autograd of its definition in 64 bits."""
    S, L, H, E, dim = t["S"], t["L"], t["H"], t["E"], t["H"] * 64
    leaf = {n: t[n].double().requires_grad_() for n in ("x", "g1", "b1", "g2", "b2", "table")}
    ek, ev = t["enc"].double().requires_grad_(), t["enc"].double().requires_grad_()

    def norm(x, g, b):
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        return (x - mean) / (var + 1e-5).sqrt() * g + b

    def att(q, k, v, mask, bias):
        x = torch.einsum("sihd,sjhd->shij", q, k) * 0.125 + bias
        return torch.einsum("shij,sjhd->sihd", torch.softmax(x.masked_fill(mask, -math.inf), -1), v)
    rel = torch.arange(L, device=DEV)[None, :] - torch.arange(L, device=DEV)[:, None]
    n1 = norm(leaf["x"], leaf["g1"], leaf["b1"]).view(S, L, H, 64)
    bias = leaf["table"][R.bucket(rel, 32, 128, False)].permute(2, 0, 1)[None]
    y = leaf["x"] + att(n1, n1, n1, (rel > 0)[None, None], bias).reshape(S * L, dim)
    n2 = norm(y, leaf["g2"], leaf["b2"]).view(S, L, H, 64)
    past = (torch.arange(E, device=DEV) >= t["klens"][:, None])[:, None, None]
    z = y + att(n2, ek, ev, past, 0.0).reshape(S * L, dim)
    names = ("x", "g1", "b1", "g2", "b2", "table")
    g = torch.autograd.grad(z, [leaf[n] for n in names] + [ek, ev], t["dz"].double().view(S * L, dim))
    return dict(zip(("z", "dx", "dg1", "db1", "dg2", "db2", "dtable", "dek", "dev"), (z.detach(),) + g))


def block_close(t, ref):
    """Norm-wise: some 10 operators of at most 2^-18 of their norm each (64-term scores, sums of up to 150 rows)."""
    for n in OUTS:
        d = (t[n].double().view(ref[n].shape) - ref[n]).norm() / ref[n].norm()
        assert float(d) <= 10 * 2.0 ** -18, (n, float(d))


def test_block_together(ctx):
    t = block_state(ctx)
    block(ctx, t)
    block_close(t, block_reference(t))


def test_graph_replays(ctx):
    """The block captured, then replayed with other inputs, eager work of the same buffers' kind between replays;
    a second graph with its own workspaces replayed beside it on another stream."""
    states, graphs = [block_state(ctx, 0), block_state(ctx, 100)], []
    for t in states:
        block(ctx, t)
    torch.cuda.synchronize()
    for t in states:
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        ctx.set_stream(s.cuda_stream)
        with torch.cuda.graph(g, stream=s):
            block(ctx, t)
        ctx.set_stream(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    other = [torch.cuda.Stream(), torch.cuda.Stream()]
    for round_ in range(4):
        want = []
        for i, t in enumerate(states):
            t["x"].copy_(randn(200 + 10 * round_ + i, *t["x"].shape))
            t["klens"].copy_(ints([t["E"] - round_, round_ + 1]))
            block(ctx, t)  # eager, in the graph's own buffers
            want.append({n: t[n].clone() for n in OUTS})
            for n in OUTS:
                t[n].fill_(NAN)
        torch.cuda.synchronize()
        for g, s in zip(graphs, other):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for t, w in zip(states, want):
            assert all(torch.equal(t[n], w[n]) for n in OUTS), round_


def test_two_streams(ctx):
    """Two contexts on two streams at once, each with its own buffers, against the same work alone."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = [native.Context(s.cuda_stream) for s in streams]
    states = [block_state(c, 50 * i, S=4, L=200, E=120) for i, c in enumerate(ctxs)]
    torch.cuda.synchronize()
    want = []
    for c, t, s in zip(ctxs, states, streams):
        with torch.cuda.stream(s):
            block(c, t)
        torch.cuda.synchronize()
        want.append({n: t[n].clone() for n in OUTS})
    torch.cuda.synchronize()
    for _ in range(3):
        for c, t, s in zip(ctxs, states, streams):
            with torch.cuda.stream(s):
                block(c, t)
    torch.cuda.synchronize()
    for t, w in zip(states, want):
        assert all(torch.equal(t[n], w[n]) for n in OUTS)
    for c in ctxs:
        c.close()


def test_timing_classes(ctx):
    t = block_state(ctx)
    ctx.timing("*")
    ctx.timing_reset()
    block(ctx, t)
    ctx.sync()
    counts = {n: ctx.timing_get(n)[1] for n in ("layernorm", "layernorm_backward", "cross_attention",
                                                "cross_attention_dq", "cross_attention_dkv")}
    ctx.timing(None)
    assert counts == {"layernorm": 2, "layernorm_backward": 2, "cross_attention": 2, "cross_attention_dq": 2,
                      "cross_attention_dkv": 2}

"""Layer norm and cross attention on the GPU: calls that are refused, and cuts of the work that other tests do not take."""

import pytest
import torch

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


def buffer(n):
    return torch.empty(max(int(n), 16), dtype=torch.uint8, device=DEV).fill_(0xff)


def make(S, H, KV, Lq, Lk, dtype=F32):
    g = torch.Generator(device=DEV)
    g.manual_seed(S + Lq)
    return [torch.randn(S, n, h, 64, device=DEV, generator=g).to(dtype) for n, h in ((Lq, H), (Lk, KV), (Lk, KV), (Lq, H))]


def test_outputs_on_inputs_refused(ctx):
    """An output that begins where another tensor does, which is read after it is written; self attention's q, k and v in
    one place are read only."""
    q, k, v, dout = make(2, 4, 4, 40, 40)
    out, table = torch.empty_like(q), torch.randn(32, 4, device=DEV)
    p = native.CrossAttention(ctx, q, k, v, out, bias_table=table)
    saved, ws = buffer(p.saved_bytes()), buffer(max(p.workspace_bytes(False), p.workspace_bytes(True)))
    before = [t.clone() for t in (q, k, v, dout)]
    for bad in (k, v):
        with pytest.raises(native.NativeError, match="address"):
            p.forward(q, k, v, bad, saved=saved, workspace=ws)
    p.forward(q, q, q, out, saved=saved, workspace=ws)
    good = dict(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v), dbias=torch.empty_like(table))
    for bad in (dict(dq=q), dict(dq=dout), dict(dq=k), dict(dq=v), dict(dk=good["dv"]), dict(dk=q), dict(dv=dout), dict(dk=dout),
                dict(dq=good["dk"]), dict(dq=k, dk=None, dv=None)):
        with pytest.raises(native.NativeError, match="address"):
            p.backward(q, k, v, out, saved, dout, workspace=ws, **{**good, **bad})
    with pytest.raises(native.NativeError, match="address"):  # k is q
        p.backward(q, q, q, out, saved, dout, dq=q, workspace=ws)
    big = buffer(p.saved_bytes() + p.workspace_bytes(True))
    with pytest.raises(native.NativeError, match="address"):
        p.backward(q, k, v, out, big, dout, workspace=big, **good)
    # q before heads, out after them: in the place of out's rows are others of dq's
    turned = torch.empty(2, 4, 40, 64, device=DEV).transpose(1, 2)
    p2 = native.CrossAttention(ctx, turned.copy_(q), k, v, out)
    with pytest.raises(native.NativeError, match="address"):
        native._ok(native.lib().vh_cross_attention(ctx.h, p2._ref, turned.data_ptr(), k.data_ptr(), v.data_ptr(),
                                                   turned.data_ptr(), None, ws.data_ptr()), "vh_cross_attention")
    p.backward(q, q, q, out, saved, dout, workspace=ws, **good)
    assert all(torch.equal(a, b) for a, b in zip((q, k, v, dout), before))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(2, 4, 2, 70, 90), (1, 4, 4, 60, 2000), (8, 16, 16, 400, 400), (1, 2, 2, 1500, 40)], ids=str)
def test_gradients_in_place(ctx, size, dtype):
    """dk on k, dv on v and dq on out; without dk and dv, dq on q or on dout; out on q: the bits of places of their own."""
    q, k, v, dout = make(*size, dtype)
    out, table = torch.empty_like(q), torch.randn(32, size[1], device=DEV)
    p = native.CrossAttention(ctx, q, k, v, out, bias_table=table, key_lengths=torch.tensor(
        [size[4] - 5 * s for s in range(size[0])], dtype=torch.int32, device=DEV), causal=size[3] == size[4])
    saved, ws = buffer(p.saved_bytes()), buffer(max(p.workspace_bytes(False), p.workspace_bytes(True)))
    p.forward(q, k, v, out, saved=saved, workspace=ws)
    want = [torch.empty_like(t) for t in (q, k, v)]
    p.backward(q, k, v, out, saved, dout, *want, workspace=ws)
    place = [t.clone() for t in (out, k, v)]
    p.backward(q, place[1], place[2], place[0], saved, dout, *place, workspace=ws)
    assert all(torch.equal(a, b) for a, b in zip(place, want))
    for i in (0, 1):
        t = [q.clone(), dout.clone()]
        p.backward(t[0], k, v, out, saved, t[1], t[i], workspace=ws)
        assert torch.equal(t[i], want[0])
    alone = torch.empty_like(q)
    p.forward(q, k, v, alone, workspace=ws)
    on_q = q.clone()
    p.forward(on_q, k, v, on_q, workspace=ws)
    assert torch.equal(on_q, alone)


def test_layernorm_in_place_at_another_pitch_refused(ctx):
    x, gamma = torch.randn(6, 16, device=DEV), torch.ones(8, device=DEV)
    stats = torch.empty(6, 2, device=DEV)
    with pytest.raises(native.NativeError, match="pitches"):
        ctx.layernorm(x, gamma, None, x, 6, 8, ldx=16, ldy=12)
    dy, ws = torch.randn(6, 16, device=DEV), buffer(1024)
    for a, b in ((dy, x), (x, dy)):
        with pytest.raises(native.NativeError, match="pitches"):
            ctx.layernorm_backward(a, b, gamma, stats, x, 6, 8, lddy=16, ldx=16, lddx=8, workspace=ws)
    ctx.layernorm(x, gamma, None, x, 1, 8, ldx=16, ldy=8)  # one row has no pitch
    ctx.layernorm(x, gamma, None, x, 6, 8, ldx=16, ldy=16, stats=stats)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("buckets", [0, 32])
@pytest.mark.parametrize("form", ["plain", "causal", "ragged"])
@pytest.mark.parametrize("size", [(8, 8, 4, 600, 256), (4, 24, 8, 1100, 250)], ids=str)
def test_shared_heads_in_pieces(ctx, size, form, buckets, dtype):
    """dk and dv of several heads in one workgroup whose queries are cut in two as well: 256 workgroups of 32 keys and from
    16 tiles of queries on, where a piece ends within one head and the next begins there."""
    S, H, KV, Lq, Lk = size
    q, k, v, dout = make(*size, dtype)
    kw = dict(causal=form == "causal")
    if form == "ragged":
        kw.update(query_lengths=[Lq - 67 * s for s in range(S)], key_lengths=[Lk - 30 * s for s in range(S)])
    if form == "causal":
        kw.update(query_start=[Lk - Lq + 9 * s for s in range(S)])
    if buckets:
        kw.update(bias_table=torch.randn(buckets, H, device=DEV), bidirectional=form != "causal")
    val, tol = R.attention(q, k, v, dout=dout, **kw)
    for n in ("query_lengths", "key_lengths", "query_start"):
        if n in kw:
            kw[n] = torch.tensor(kw[n], dtype=torch.int32, device=DEV)
    got = {"out": torch.empty_like(q)}
    p = native.CrossAttention(ctx, q, k, v, got["out"], **kw)
    saved, ws = buffer(p.saved_bytes()), buffer(max(p.workspace_bytes(False), p.workspace_bytes(True)))
    p.forward(q, k, v, got["out"], saved=saved, workspace=ws)
    got.update(dq=torch.empty_like(q), dk=torch.empty_like(k), dv=torch.empty_like(v))
    if buckets:
        got["dbias"] = torch.empty_like(kw["bias_table"])
    ws.fill_(0xff)
    p.backward(q, k, v, got["out"], saved, dout, got["dq"], got["dk"], got["dv"], dbias=got.get("dbias"), workspace=ws)
    for n in got:
        R.assert_within(got[n], val[n], tol[n], f"{size} {form} {n}")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("size", [(1, 4, 2, 100, 3000), (2, 4, 2, 70, 90), (4, 12, 12, 1030, 64)], ids=str)
def test_table_without_gradient(ctx, size, dtype):
    """A table whose gradient is not wanted, also where it would be joined from pieces: the other gradients keep their bits."""
    q, k, v, dout = make(*size, dtype)
    table, out = torch.randn(32, size[1], device=DEV), torch.empty_like(q)
    p = native.CrossAttention(ctx, q, k, v, out, bias_table=table)
    saved, ws = buffer(p.saved_bytes()), buffer(max(p.workspace_bytes(False), p.workspace_bytes(True)))
    p.forward(q, k, v, out, saved=saved, workspace=ws)
    r = []
    for dbias in (torch.empty_like(table), None):
        g = [torch.empty_like(t) for t in (q, k, v)]
        p.backward(q, k, v, out, saved, dout, *g, dbias=dbias, workspace=ws)
        r.append(g)
    assert all(torch.equal(a, b) for a, b in zip(*r)) and all(bool(t.isfinite().all()) for t in r[0])

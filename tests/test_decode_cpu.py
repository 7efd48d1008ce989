"""Rotary positions, the paged cache and beam search without a GPU: refusals, sizes, the bindings' checks, and the definitions
that the GPU tests compare with."""

import ctypes
import math

import pytest
import torch

import decode_ref as R
from vocalarc_hip import native

pytestmark = pytest.mark.skipif(not native.LIB_PATH.exists(), reason="library not built")
NULL = ctypes.c_void_p(None)


def change(c, **fields):
    for name, value in fields.items():
        if isinstance(value, tuple):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def cache(**fields):
    return change(native.CCache(1, 2, 64, 32, 10, 3, 5), **fields)


def queries(**fields):
    return change(native.CCacheQueries(0, 4, 7, 0, 100, 0.125, (7 * 256, 256, 64), (7 * 256, 256, 64)), **fields)


def beam(**fields):
    return change(native.CBeam(0, 2, 3, 50, 4, -1, (150, 50)), **fields)


def refused(n, text):
    assert n == 0 and text in native.last_error(), (n, native.last_error())


@pytest.mark.parametrize("fields,text", [
    ({"type": 2}, "type"), ({"kv_heads": 0}, "heads"), ({"kv_heads": 4097}, "heads"), ({"head_dim": 96}, "heads"),
    ({"page_tokens": 0}, "pages"), ({"page_tokens": 24}, "pages"), ({"page_tokens": 4112}, "pages"), ({"pages": 0}, "pages"),
    ({"sequences": -1}, "table"), ({"sequences": (1 << 20) + 1}, "table"), ({"table_pages": -1}, "table"),
    ({"table_pages": (1 << 24) + 1}, "table"), ({"kv_heads": 4096, "page_tokens": 4096, "head_dim": 128}, "bytes"),
    ({"kv_heads": 4096, "page_tokens": 2032, "pages": 1 << 30}, "bytes"),
])
def test_cache_refused(fields, text):
    refused(native.lib().vh_cache_bytes(ctypes.byref(cache(**fields))), text)
    refused(native.lib().vh_cache_workspace_bytes(ctypes.byref(cache(**fields)), ctypes.byref(queries())), text)


def test_cache_sizes():
    for kind, element in ((0, 2), (1, 1)):
        for kv, dim, page, pages in ((1, 64, 16, 1), (3, 128, 48, 7), (8, 128, 4096, 1000)):
            n = native.lib().vh_cache_bytes(ctypes.byref(cache(type=kind, kv_heads=kv, head_dim=dim, page_tokens=page, pages=pages)))
            values = pages * page * kv * dim * 2 * element
            scales = pages * page // 16 * kv * 8 * kind
            assert values + scales <= n <= values + scales + 256 * pages and n % (256 * pages) == 0
    assert native.lib().vh_cache_bytes(ctypes.byref(cache(sequences=0, table_pages=0))) > 0


@pytest.mark.parametrize("fields,text", [
    ({"type": 2}, "type"), ({"heads": 0}, "heads"), ({"heads": 3}, "heads"), ({"heads": 65538}, "heads"), ({"length": -1}, "length"),
    ({"length": (1 << 29) + 1}, "length"), ({"heads": 64, "length": 1 << 27}, "length"), ({"most_keys": -1}, "keys"),
    ({"scale": math.nan}, "scale"), ({"scale": math.inf}, "scale"), ({"q_strides": (1792, 254, 64)}, "q's strides"),
    ({"q_strides": (1792, 256, -64)}, "q's strides"), ({"q_strides": (1792, 1 << 25, 64)}, "q's strides"),
    ({"out_strides": (1792, 256, 32)}, "overlap"), ({"out_strides": (0, 256, 64)}, "overlap"),
])
def test_queries_refused(fields, text):
    refused(native.lib().vh_cache_workspace_bytes(ctypes.byref(cache()), ctypes.byref(queries(**fields))), text)


def test_queries_taken():
    for fields in ({}, {"length": 0}, {"most_keys": 0}, {"type": 1}, {"q_strides": (0, 0, 0)}, {"length": 1, "out_strides": (256, -5, 64)},
                   {"scale": 0.0}, {"scale": -1.0}):
        assert native.lib().vh_cache_workspace_bytes(ctypes.byref(cache()), ctypes.byref(queries(**fields))) >= 16, native.last_error()
    assert native.lib().vh_cache_workspace_bytes(ctypes.byref(cache(sequences=0)), ctypes.byref(queries())) >= 16


def test_workspace_of_pieces():
    """Long caches of few rows take room for pieces: of D + 2 floats a row each."""
    c = cache(sequences=1, table_pages=4096, head_dim=128)
    n = native.lib().vh_cache_workspace_bytes(ctypes.byref(c), ctypes.byref(queries(length=1, most_keys=100_000, out_strides=(512, 512, 128))))
    assert n > 16 and n % (4 * 130 * 4) == 0


@pytest.mark.parametrize("fields,text", [
    ({"type": 3}, "type"), ({"sequences": -1}, "sequences"), ({"beams": 0}, "beams"), ({"beams": 65}, "beams"), ({"vocab": 0}, "tokens"),
    ({"vocab": (1 << 24) + 1}, "tokens"), ({"picks": 0}, "picks"), ({"picks": 65}, "picks"), ({"vocab": 1, "picks": 4}, "picks"),
    ({"end_token": -2}, "end token"), ({"end_token": 50}, "end token"), ({"strides": (-1, 50)}, "strides"),
    ({"strides": (150, -1)}, "strides"),
])
def test_beam_refused(fields, text):
    refused(native.lib().vh_beam_workspace_bytes(ctypes.byref(beam(**fields))), text)


def test_beam_sizes():
    one = native.lib().vh_beam_workspace_bytes(ctypes.byref(beam()))
    assert one >= 6 * (16 + 4 * 8)
    for kind in (0, 1):
        n = native.lib().vh_beam_workspace_bytes(ctypes.byref(beam(type=kind, sequences=64, beams=16, vocab=1 << 24, picks=64)))
        assert n >= 64 * 16 * 256 * 64 * 8
    assert native.lib().vh_beam_workspace_bytes(ctypes.byref(beam(sequences=0))) == 16
    assert native.lib().vh_beam_workspace_bytes(ctypes.byref(beam(sequences=1, beams=1, strides=(-3, -4)))) >= 16


def test_null_arguments():
    L = native.lib()
    c, q, r, b = cache(), queries(), native.CRotary(64, 0, 5, 16), beam()
    for n in (L.vh_rotary_table(None, None, 2, 1, None), L.vh_rotary_apply(None, ctypes.byref(r), None, None, None, 0),
              L.vh_cache_append(None, ctypes.byref(c), None, None, None, None), L.vh_cache_read(None, ctypes.byref(c), None, None, None),
              L.vh_cache_attention(None, ctypes.byref(c), ctypes.byref(q), None, None, None, None),
              L.vh_cache_reorder(None, ctypes.byref(c), 1, *[None] * 5), L.vh_beam_select(None, ctypes.byref(b), *[None] * 8)):
        refused(n, "null context")
    refused(L.vh_cache_bytes(None), "null cache")
    refused(L.vh_cache_workspace_bytes(ctypes.byref(c), None), "null queries")
    refused(L.vh_beam_workspace_bytes(None), "null beam")


def plans(kind="int8"):
    pool = native.PagedCache(None, kind, kv_heads=2, head_dim=64, page_tokens=32, pages=10, device="cpu")
    return pool, torch.zeros(3, 5, dtype=torch.int32), torch.zeros(3, 7, 2, 64), torch.zeros(3, 7, 4, 64)


def test_binding_checks_layouts():
    pool, table, k, q = plans()
    i3, bad = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    with pytest.raises(native.NativeError, match="bf16 or int8"):
        native.PagedCache(None, "fp8", kv_heads=2, head_dim=64, page_tokens=32, pages=10, device="cpu")
    with pytest.raises(native.NativeError, match="unsupported cache"):
        native.PagedCache(None, "int8", kv_heads=2, head_dim=80, page_tokens=32, pages=10, device="cpu")
    for t in (table.long(), table[0], table.t(), table.to("meta")):
        with pytest.raises(native.NativeError):
            pool.tokens(t, k, k)
    for kk, vv in ((k[:2], k[:2]), (k, k[:, :3]), (k[:, :, :1], k[:, :, :1]), (k.double(), k.double()), (k, k.bfloat16()),
                   (torch.zeros(3, 7, 2, 128)[..., ::2], k)):
        with pytest.raises(native.NativeError):
            pool.tokens(table, kk, vv)
    for more in ({"start": bad}, {"lengths": i3[:2]}, {"start": i3.to("meta")}):
        with pytest.raises(native.NativeError):
            pool.tokens(table, k, k, **more)
    for qq, out in ((q[:2], q[:2]), (q, q[:, :3]), (q, q.bfloat16()), (torch.zeros(3, 7, 4, 32),) * 2):
        with pytest.raises(native.NativeError):
            pool.queries(table, qq, out, most_keys=5)
    for more in ({"key_lengths": bad}, {"query_lengths": i3[:2]}, {"query_start": bad}):
        with pytest.raises(native.NativeError):
            pool.queries(table, q, q, most_keys=5, **more)
    with pytest.raises(native.NativeError):
        native.BeamSearch(None, torch.zeros(2, 50))
    with pytest.raises(native.NativeError):
        native.BeamSearch(None, torch.zeros(2, 3, 50, dtype=torch.float16))
    c = pool.queries(table, q, q, most_keys=5, causal=True).c
    assert (c.sequences, c.table_pages, c.kv_heads, c.pages) == (3, 5, 2, 10)


def test_binding_checks_calls():
    """Tensors of other layouts, buffers that are too small, and tensors that the context's GPU cannot read."""
    pool, table, k, q = plans("bf16")
    t, p = pool.tokens(table, k, k), pool.queries(table, q, q, most_keys=5)
    for args, text in (((k[:2], k), "k is not"), ((k, k.bfloat16()), "v is not"), ((k.transpose(1, 2), k), "k is not"), ((k, k), "cpu")):
        with pytest.raises(native.NativeError, match=text):
            t.append(*args)
        with pytest.raises(native.NativeError, match=text):
            t.read(*args)
    ws = torch.zeros(p.workspace_bytes(), dtype=torch.uint8)
    for args, w, text in (((q[:2], q), ws, "q is not"), ((q, q.double()), ws, "out is not"), ((q, q), ws[1:], "workspace"),
                          ((q, q), ws[:1].expand(ws.numel()), "workspace"), ((q, q), ws, "cpu")):
        with pytest.raises(native.NativeError, match=text):
            p.forward(*args, workspace=w)
    i3 = torch.zeros(3, dtype=torch.int32)
    good = dict(table=table, parents=i3, lengths=i3[:1], spare=i3, table_out=table, spare_out=i3, beams=3)
    for more, text in (({"beams": 2}, "groups"), ({"beams": 0}, "groups"), ({"parents": i3[:2]}, "parents"), ({"lengths": i3}, "lengths"),
                       ({"spare": i3.long()}, "spare"), ({"table_out": table[:2]}, "table_out"), ({"spare_out": i3[:1]}, "spare_out"),
                       ({}, "cpu")):
        with pytest.raises(native.NativeError, match=text):
            pool.reorder(**{**good, **more})
    x = torch.zeros(2, 3, 50)
    b = native.BeamSearch(None, x, picks=4, end_token=1)
    ws = torch.zeros(b.workspace_bytes(), dtype=torch.uint8)
    i, f = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 4)
    good = dict(logits=x, scores=f[:, :3].contiguous(), tokens=i, parents=i, new_scores=f, ended=i[:, :3].contiguous(), new_ended=i,
                workspace=ws)
    for more, text in (({"logits": x.bfloat16()}, "logits"), ({"scores": f}, "scores"), ({"tokens": i.long()}, "tokens"),
                       ({"parents": i[:, :2]}, "parents"), ({"new_scores": f.double()}, "new_scores"), ({"ended": i}, "ended"),
                       ({"new_ended": i[:1]}, "new_ended"), ({"workspace": ws[1:]}, "workspace"), ({}, "cpu")):
        with pytest.raises(native.NativeError, match=text):
            b.select(**{**good, **more})


def test_binding_refuses_rotations():
    for positions, dim in ((0, 4), (5, 3), (5, 0), (5, 258)):
        with pytest.raises(native.NativeError, match="positions"):
            native.Rotary(None, positions, dim)


# ---------------------------------------------------------------- the definitions against each other

@pytest.mark.parametrize("interleaved", [False, True])
def test_reference_rotation(interleaved):
    """Complex numbers; the transpose undoes it; the step-by-step form is within its bound."""
    x = torch.randn(2, 5, 3, 24, generator=torch.Generator().manual_seed(0))
    val, tol = R.rotary(x, [0, 100], 16, interleaved)
    back, _ = R.rotary(val, [0, 100], 16, interleaved, backward=True)
    assert (back - x.double()).abs().max() < 1e-12
    z = (x[..., 0:16:2], x[..., 1:16:2]) if interleaved else (x[..., :8], x[..., 8:16])
    z = torch.complex(z[0].double(), z[1].double())
    p = torch.tensor([0, 100])[:, None] + torch.arange(5)
    z = z * torch.polar(torch.ones(8, dtype=torch.float64), p[..., None, None] * R.theta(16))
    got = torch.complex(val[..., 0:16:2], val[..., 1:16:2]) if interleaved else torch.complex(val[..., :8], val[..., 8:16])
    assert (got - z).abs().max() < 1e-12
    table = torch.stack(((torch.arange(200)[:, None] * R.theta(16)).cos(), (torch.arange(200)[:, None] * R.theta(16)).sin()), -1).float()
    for s, a in enumerate((0, 100)):
        R.assert_within(R.turn32(x[s], table, a, interleaved), val[s], tol[s], "turn32")


def test_reference_cache():
    """A block's tokens by ones and all at once stand for the rows to within the steps that they were rounded in."""
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn(40, 2, 8, generator=g), torch.randn(40, 2, 8, generator=g)
    a, b = R.Cache("int8", 1, 2, 8), R.Cache("int8", 1, 2, 8)
    a.append(0, 0, k, v)
    for t in range(40):
        b.append(0, t, k[t:t + 1], v[t:t + 1])
    for c, steps in ((a, 1), (b, 16)):
        for part, x in enumerate((k, v)):
            step = c.s[0][part].repeat_interleave(16, 0)[:40, :, None]
            assert ((c.values(0, part) - x).abs() <= step * steps * 0.5001).all()
    assert torch.allclose(a.s[0][0], b.s[0][0], rtol=1e-6)


def test_reference_beams():
    x = torch.randn(3, 20, generator=torch.Generator().manual_seed(2))
    s = torch.tensor([-1.0, -2.0, -0.5])
    want = (torch.log_softmax(x.double(), -1) + s.double()[:, None]).flatten().sort(descending=True)
    got, _ = R.beams(x, s, 6)
    assert [b * 20 + t for _, b, t in got] == want.indices[:6].tolist()
    assert max(abs(v - w) for (v, _, _), w in zip(got, want.values.tolist())) < 1e-12

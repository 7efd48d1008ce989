"""Layer norm and cross attention without a GPU: refusals, sizes and the bias's buckets."""

import ctypes

import pytest
import torch

import norm_cross_ref as R
from vocalarc_hip import native

pytestmark = pytest.mark.skipif(not native.LIB_PATH.exists(), reason="library not built")


def layout(**change):
    c = native.CCross(0, 2, 8, 4, 5, 7, 0, 0.125)
    c.q_strides[:] = c.out_strides[:] = (5 * 512, 512, 64)
    c.k_strides[:] = c.v_strides[:] = (7 * 256, 256, 64)
    for name, value in change.items():
        if isinstance(value, tuple):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def refused(c, backward, text):
    n = native.lib().vh_cross_workspace_bytes(ctypes.byref(c), backward)
    assert n == 0 and text in native.last_error(), (n, native.last_error())
    return True


@pytest.mark.parametrize("change,text", [
    ({"type": 2}, "type"), ({"sequences": -1}, "sequences"), ({"heads": 0}, "heads"), ({"kv_heads": 0}, "heads"),
    ({"kv_heads": 3}, "heads"), ({"query_length": -1}, "lengths"), ({"key_length": -1}, "lengths"),
    ({"key_length": (1 << 29) + 1}, "lengths"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
    ({"q_strides": (2560, 510, 64)}, "q's strides"), ({"k_strides": (1792, 256, 2)}, "k's strides"),
    ({"v_strides": (-1792, 256, 64)}, "v's strides"), ({"v_strides": (1792, 1 << 25, 64)}, "row stride"),
    ({"out_strides": (0, 512, 64)}, "overlap"), ({"out_strides": (2560, 512, 32)}, "overlap"),
    ({"out_strides": (2048, 512, 64)}, "overlap"),
    ({"bias_table": 16, "buckets": 1, "max_distance": 128}, "buckets"),
    ({"bias_table": 16, "buckets": 130, "max_distance": 128}, "buckets"),
    ({"bias_table": 16, "buckets": 31, "max_distance": 128, "bidirectional": 1}, "buckets"),
    ({"bias_table": 16, "buckets": 2, "max_distance": 128, "bidirectional": 1}, "buckets"),
    ({"bias_table": 16, "buckets": 32, "max_distance": 16}, "buckets"),
    ({"bias_table": 16, "buckets": 32, "max_distance": 4097}, "buckets"),
    ({"sequences": 1 << 20, "heads": 1 << 12, "kv_heads": 1, "query_length": 1, "key_length": 1,
      "q_strides": (1 << 18, 64, 64), "out_strides": (1 << 18, 64, 64)}, "workgroups"),
])
def test_layout_refused(change, text):
    assert refused(layout(**change), 0, text)


@pytest.mark.parametrize("change,backward", [
    # single rows of 2^24 (sequence, head) pairs, a workgroup each; more key tiles than that beside single queries
    ({"sequences": 1 << 20, "heads": 16, "kv_heads": 16, "query_length": 1, "key_length": 1}, 0),
    ({"sequences": 1 << 21, "heads": 1, "kv_heads": 1, "query_length": 1, "key_length": 1025}, 1),
])
def test_launches_beyond_the_device(change, backward):
    heads = change["heads"] * 64
    rows = (change["query_length"] * heads, heads, 64)
    c = layout(**change, q_strides=rows, out_strides=rows, k_strides=(change["key_length"] * heads, heads, 64),
               v_strides=(change["key_length"] * heads, heads, 64))
    assert refused(c, backward, "workgroups")
    c.sequences //= 2
    assert native.lib().vh_cross_workspace_bytes(ctypes.byref(c), backward) > 0, native.last_error()


def test_strides_of_single_ones():
    """Where there is one sequence, row or head, its stride counts for nothing."""
    odd = (7, -3, 1 << 60)
    c = layout(sequences=1, heads=1, kv_heads=1, query_length=1, key_length=1, q_strides=odd, k_strides=odd, v_strides=odd,
               out_strides=odd)
    assert native.lib().vh_cross_workspace_bytes(ctypes.byref(c), 1) > 0, native.last_error()


def test_broadcast_inputs_have_no_gradient():
    """Keys that all sequences share, or heads on one place: fine to read, refused where a gradient goes there."""
    for name, strides in (("k_strides", (0, 256, 64)), ("v_strides", (1792, 0, 64)), ("q_strides", (2560, 512, 0))):
        c = layout(**{name: strides})
        assert native.lib().vh_cross_workspace_bytes(ctypes.byref(c), 0) > 0
        assert refused(c, 1, "overlap")


def test_layouts_taken():
    for change in ({}, {"sequences": 0}, {"query_length": 0}, {"key_length": 0}, {"type": 1},
                   {"q_strides": (2560, 64, 320), "out_strides": (2560, 64, 320)},  # [S][H][L][64]
                   {"q_strides": (64, 1024, 128), "out_strides": (64, 1024, 128)},  # rows outermost
                   {"bias_table": 16, "buckets": 2, "max_distance": 2},
                   {"bias_table": 16, "buckets": 4, "max_distance": 2, "bidirectional": 1},
                   {"bias_table": 16, "buckets": 128, "max_distance": 4096}):
        c = layout(**change)
        for backward in (0, 1):
            assert native.lib().vh_cross_workspace_bytes(ctypes.byref(c), backward) > 0, (change, native.last_error())
        assert native.lib().vh_cross_saved_bytes(ctypes.byref(c)) > 0


def test_null_context_and_layout():
    L = native.lib()
    c = layout()
    assert not L.vh_cross_attention(None, ctypes.byref(c), None, None, None, None, None, None)
    assert "null context" in native.last_error()
    assert not L.vh_cross_attention_backward(None, ctypes.byref(c), *[None] * 11)
    assert not L.vh_layernorm(None, 0, 1, 4, None, 4, None, None, 1e-5, None, 4, None)
    assert not L.vh_layernorm_backward(None, 0, 1, 4, None, 4, None, 4, None, None, None, 4, None, None, None)
    assert not L.vh_cross_workspace_bytes(None, 0) and "null layout" in native.last_error()


@pytest.mark.parametrize("rows,dim", [(-1, 4), (1 << 31, 4), (1, 0), (1, 16385)])
def test_layernorm_refused(rows, dim):
    with pytest.raises(native.NativeError, match="unsupported"):
        native.Context.layernorm_workspace_bytes(rows, dim)


def test_layernorm_workspace():
    # the backward pass's workgroups, a row of dgamma and one of dbeta each
    assert native.Context.layernorm_workspace_bytes(0, 1) >= 16
    for rows, dim in ((1, 1), (7, 384), (49662, 384), (3, 16384), (100000, 2048)):
        n = native.Context.layernorm_workspace_bytes(rows, dim)
        assert 8 * dim <= n <= 8 * dim * 512 and n % (8 * dim) == 0


@pytest.mark.parametrize("bidirectional", [0, 1])
@pytest.mark.parametrize("buckets,max_distance", [(32, 128), (16, 96), (64, 800), (4, 2), (4, 7), (128, 4096), (6, 27),
                                                  (32, 256), (20, 1000), (128, 65), (8, 64)])
def test_buckets(buckets, max_distance, bidirectional):
    """Every distance, the borders' own among them (16 of 8 to 128 in 8 steps meets them in whole numbers)."""
    if max_distance <= (buckets // 2 if bidirectional else buckets) // 2:  # no distance left for the far buckets
        assert native.lib().vh_relative_bucket(1, buckets, max_distance, bidirectional) == -1
        return
    far = max_distance + 40
    rel = torch.arange(-far, far + 1)
    want = R.bucket(rel, buckets, max_distance, bool(bidirectional))
    got = [native.lib().vh_relative_bucket(int(r), buckets, max_distance, bidirectional) for r in rel]
    assert got == want.tolist()
    for r in (-2 ** 31, 2 ** 31 - 1):
        assert native.lib().vh_relative_bucket(r, buckets, max_distance, bidirectional) == \
            int(want[0] if r < 0 else want[-1])


def test_bucket_refused():
    for args in ((0, 1, 128, 0), (0, 33, 128, 1), (0, 32, 8, 1), (0, 32, 5000, 1)):
        assert native.lib().vh_relative_bucket(*args) == -1 and "buckets" in native.last_error()


def test_binding_checks_shapes():
    q, k = torch.zeros(2, 5, 8, 64), torch.zeros(2, 7, 4, 64)
    table = torch.zeros(32, 8)
    good = dict(q=q, k=k, v=k, out=q)
    for bad in ({"q": q[..., :32]}, {"v": k[:, :3]}, {"k": k.bfloat16()}, {"out": q[:, :4]}, {"k": k[:1], "v": k[:1]},
                {"q": q.double(), "k": k.double(), "v": k.double(), "out": q.double()},
                {"q": torch.zeros(2, 5, 8, 128)[..., ::2]},
                {"key_lengths": torch.zeros(2)}, {"key_lengths": torch.zeros(3, dtype=torch.int32)},
                {"bias_table": table[:, :4]}, {"bias_table": table.double()}):
        with pytest.raises(native.NativeError):
            native.CrossAttention(None, **{**good, **bad})
    c = native.CrossAttention(None, **good, bias_table=table).c
    assert (c.sequences, c.heads, c.kv_heads, c.query_length, c.key_length, c.buckets) == (2, 8, 4, 5, 7, 32)
    assert list(c.k_strides) == [7 * 256, 256, 64]


def test_binding_checks_calls():
    """Tensors of a later call that the layout does not describe, and buffers that are too small, are refused before the
    library sees them."""
    q, k = torch.zeros(2, 5, 8, 64), torch.zeros(2, 7, 4, 64)
    table = torch.zeros(32, 8)
    p = native.CrossAttention(None, q, k, k, q, bias_table=table)
    saved, ws = torch.zeros(p.saved_bytes(), dtype=torch.uint8), torch.zeros(p.workspace_bytes(True), dtype=torch.uint8)
    good = dict(q=q, k=k, v=k, out=q, saved=saved, workspace=ws)
    more = dict(dout=q, dq=q, dk=k, dv=k, dbias=table)
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    for bad, text in (({"q": turned}, "q is not"), ({"k": k.bfloat16()}, "k is not"), ({"v": k[:, :5]}, "v is not"),
                      ({"out": turned}, "out is not"), ({"saved": saved[:-1]}, "saved"), ({"workspace": ws[:15]}, "workspace")):
        with pytest.raises(native.NativeError, match=text):
            p.forward(**{**good, **bad})
    for bad, text in (({"dout": q[:1, :1].expand_as(q)}, "dout is not"), ({"dq": turned}, "dq is not"),
                      ({"dk": k[:1]}, "dk is not"), ({"dv": k.double()}, "dv is not"), ({"workspace": ws[:-1]}, "workspace"),
                      ({"saved": saved[:-1]}, "saved"), ({"dbias": table[:16]}, "dbias"), ({"dbias": table.t()}, "dbias"),
                      ({"dbias": table.bfloat16()}, "dbias")):
        with pytest.raises(native.NativeError, match=text):
            p.backward(**{**good, **more, **bad})
    with pytest.raises(native.NativeError, match="devices"):
        native.CrossAttention(None, q, k, k, q, bias_table=table.to("meta"))


def test_binding_refuses_reordered_tensors():
    """Contiguous tensors of as many elements are taken where their shape joins or splits neighbouring dimensions, not
    where it has them in another order (heads before rows)."""
    q, k = torch.zeros(2, 5, 8, 64), torch.zeros(2, 7, 4, 64)
    p = native.CrossAttention(None, q, k, k, q)
    for shape in ((10, 512), (2, 5, 512), (10, 8, 64), (5120,), (1, 10, 512), (2, 5, 4, 2, 64), (2, 5, 8, 2, 32), (2, 40, 2, 32)):
        assert p._tensor("q", "q", torch.zeros(shape)), shape
    for shape in ((2, 8, 5, 64), (16, 5, 64), (16, 320), (2, 8, 320), (5, 2, 8, 64), (2, 5, 64, 8), (8, 2, 5, 64), (40, 128),
                  (4, 20, 64), (2, 10, 4, 64)):
        with pytest.raises(native.NativeError, match="q is not"):
            p._tensor("q", "q", torch.zeros(shape))
    with pytest.raises(native.NativeError, match="k is not"):
        p.forward(q, torch.zeros(2, 4, 7, 64), k, q)
    with pytest.raises(native.NativeError, match="dv is not"):
        saved, ws = torch.zeros(p.saved_bytes(), dtype=torch.uint8), torch.zeros(p.workspace_bytes(True), dtype=torch.uint8)
        p.backward(q, k, k, q, saved, q, q, k, torch.zeros(2, 4, 7, 64), workspace=ws)
    empty = native.CrossAttention(None, q[:0], k[:0], k[:0], q[:0])
    empty._tensor("q", "q", torch.zeros(0, 8, 5, 64))


def test_binding_refuses_buffers_in_pieces():
    """A buffer's elements are counted only where they lie one behind the other."""
    q, k = torch.zeros(2, 5, 8, 64), torch.zeros(2, 7, 4, 64)
    p = native.CrossAttention(None, q, k, k, q)
    n, w = p.saved_bytes(), p.workspace_bytes(True)
    byte = torch.zeros(1, dtype=torch.uint8)
    for bad in (byte.expand(n), torch.zeros(2 * n, dtype=torch.uint8)[::2]):
        with pytest.raises(native.NativeError, match="saved"):
            p.forward(q, k, k, q, saved=bad)
    with pytest.raises(native.NativeError, match="workspace"):
        p.forward(q, k, k, q, workspace=byte.expand(w))
    with pytest.raises(native.NativeError, match="workspace"):
        p.backward(q, k, k, q, torch.zeros(n, dtype=torch.uint8), q, q, workspace=byte.expand(w))


def test_binding_refuses_other_devices():
    """Calls whose tensors the context's GPU cannot read: host memory, another GPU's."""
    q, k = torch.zeros(2, 5, 8, 64), torch.zeros(2, 7, 4, 64)
    p = native.CrossAttention(None, q, k, k, q)
    saved, ws = torch.zeros(p.saved_bytes(), dtype=torch.uint8), torch.zeros(p.workspace_bytes(True), dtype=torch.uint8)
    with pytest.raises(native.NativeError, match="cpu"):
        p.forward(q, k, k, q, workspace=ws)
    with pytest.raises(native.NativeError, match="cpu"):
        p.backward(q, k, k, q, saved, q, q, k, k, workspace=ws)


def test_sizes_whose_products_pass_64_bits():
    """2^30 sequences x 2^16 heads x 2^18 tiles are 2^64 workgroups, which is none in 64 bits; 2^45 elements between 2^20
    heads leave no room for a second sequence 2^46 behind the first."""
    c = layout(sequences=1 << 30, heads=1 << 16, kv_heads=1, query_length=1, key_length=((1 << 18) - 1) * 128,
               q_strides=(1 << 22, 64, 64), out_strides=(1 << 22, 64, 64), k_strides=(0, 64, 64), v_strides=(0, 64, 64))
    assert native.lib().vh_cross_saved_bytes(ctypes.byref(c)) == 0 and "workgroups" in native.last_error()
    c = layout(sequences=2, heads=1 << 16, kv_heads=1, query_length=1, out_strides=(1 << 46, 64, 1 << 45))
    assert native.lib().vh_cross_saved_bytes(ctypes.byref(c)) == 0 and "overlap" in native.last_error()
    c = layout(sequences=1 << 20, heads=2, kv_heads=1, query_length=1, out_strides=(1 << 45, 64, 1 << 46))
    assert native.lib().vh_cross_saved_bytes(ctypes.byref(c)) == 0 and "overlap" in native.last_error()

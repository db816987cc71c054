"""The paged cache's host side: sizes and the checks before any launch (no GPU)."""
import ctypes

import pytest


def shape(fm, **kw):
    d = dict(layers=2, kv_heads=8, head_dim=256, page_size=32, bits=16, num_pages=10, max_seqs=4, max_blocks=6)
    d.update(kw)
    c = fm.paged.PagedKvC(*(d[k] for k in ("layers", "kv_heads", "head_dim", "page_size", "bits", "num_pages",
                                            "max_seqs", "max_blocks")))
    base = 1 << 40  # never dereferenced
    c.pages = c.table = c.lens = c.refs = c.refused = base
    return c


@pytest.mark.parametrize("bits,dim,row", [(16, 256, 512), (16, 512, 1024), (4, 256, 144), (4, 512, 288)])
def test_pool_bytes(fm, bits, dim, row):
    c = shape(fm, bits=bits, head_dim=dim)
    assert fm.lib().fmoe_paged_bytes(ctypes.byref(c)) == 2 * 10 * 8 * 2 * 32 * row
    assert fm.lib().fmoe_paged_workspace_bytes(ctypes.byref(c)) > 0


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=128), -5), (dict(bits=8), -5), (dict(page_size=48), -5), (dict(page_size=0), -5), (dict(layers=0), -1),
    (dict(num_pages=0), -1), (dict(max_seqs=-1), -1), (dict(max_blocks=0), -1), (dict(kv_heads=0), -1),
    (dict(max_blocks=1 << 30), -1), (dict(num_pages=1 << 22), -1),
])
def test_shapes_refused(fm, kw, code):
    c = shape(fm, **kw)
    assert fm.lib().fmoe_paged_bytes(ctypes.byref(c)) == 0
    assert fm.lib().fmoe_paged_free(ctypes.byref(c), None, 0, None) == code


def test_pointers_and_counts_refused(fm):
    L, base = fm.lib(), 1 << 40
    c = shape(fm)
    r = ctypes.byref(c)
    ws = L.fmoe_paged_workspace_bytes(r)
    assert L.fmoe_paged_free(None, base, 1, None) == -1
    assert L.fmoe_paged_free(r, base, 5, None) == -1 and "5 sequences of 4" in fm.last_error()
    assert L.fmoe_paged_free(r, None, 1, None) == -1
    assert L.fmoe_paged_free(r, None, 0, None) == 0
    assert L.fmoe_paged_trim(r, base, 1, 0, 0, None) == -1
    assert L.fmoe_paged_reserve(r, base, base, 1, base, base, ws - 1, None) == -3
    assert L.fmoe_paged_reserve(r, base, base, 1, None, base, ws, None) == -1
    assert L.fmoe_paged_fork(r, base, None, 1, base, ws, None) == -1
    assert L.fmoe_paged_fork(r, base, base, 1, None, ws, None) == -3
    assert L.fmoe_paged_compact(r, None, base, ws, None) == -1
    assert L.fmoe_paged_copy(r, base, base, 11, None) == -1
    for field in ("pages", "table", "lens", "refs", "refused"):
        d = shape(fm)
        setattr(d, field, None)
        assert L.fmoe_paged_free(ctypes.byref(d), base, 1, None) in (-1, -2)
    d = shape(fm)
    d.pages = base + 64
    assert L.fmoe_paged_free(ctypes.byref(d), base, 1, None) == -2


def test_row_calls_refused(fm):
    L, base = fm.lib(), 1 << 40
    r = ctypes.byref(shape(fm))
    b = fm.paged.PagedBatchC(2, 1, 2, base, base, base)
    rb = ctypes.byref(b)
    norm = fm.paged.QKNormRopeC(base, base, 1e-6, 1e4, 256)
    need = L.fmoe_paged_attend_workspace_bytes(r, 16, 2, 2, 1)
    assert need > 0 and L.fmoe_paged_attend_workspace_bytes(r, 12, 2, 2, 1) == 0
    W = 8 * 256
    attend = lambda layer=0, q=base, qs=2 * W, heads=16, batch=rb, win=0, sinks=0, sc=1.0, out=base, ws=base, n=need: \
        L.fmoe_paged_attend(r, layer, q, qs, heads, batch, win, sinks, sc, out, ws, n, None)  # noqa: E731
    assert attend(layer=2) == -1 and attend(layer=-1) == -1 and attend(heads=12) == -5 and attend(heads=72) == -5
    assert attend(q=None) == -2 and attend(q=base + 8) == -2 and attend(out=base + 2) == -2 and attend(qs=2 * W + 4) == -2
    assert attend(qs=W) == -2 and attend(win=-1) == -1 and attend(sinks=-1) == -1 and attend(sc=float("inf")) == -1
    assert attend(ws=None) == -3 and attend(n=need - 1) == -3 and attend(batch=None) == -1
    for bad in (fm.paged.PagedBatchC(-1, 1, 2, base, base, base), fm.paged.PagedBatchC(2, -1, 2, base, base, base),
                fm.paged.PagedBatchC(2, 1, 1 << 40, base, base, base), fm.paged.PagedBatchC(2, 1, 2, None, base, base)):
        assert attend(batch=ctypes.byref(bad)) == -1
    assert attend(batch=ctypes.byref(fm.paged.PagedBatchC(0, 0, 0, None, None, None))) == 0
    app = lambda k=base, ks=W, v=base, vs=W, layer=0: L.fmoe_paged_append(r, layer, k, ks, v, vs, rb, None)  # noqa: E731
    assert app(k=None) == -2 and app(v=base + 4) == -2 and app(ks=W - 8) == -2 and app(vs=W + 1) == -2 and app(layer=2) == -1
    qkv = lambda n=norm, heads=16, qo=base, q=base, qs=2 * W: \
        L.fmoe_paged_append_qkv(r, 0, q, qs, heads, base, W, None, 0, rb, ctypes.byref(n) if n else None, qo, None)  # noqa: E731
    assert qkv(n=None) == -2 and qkv(heads=0) == -1 and qkv(qo=None) == -2 and qkv(q=None) == -2 and qkv(qs=W) == -2
    for f, v, code in (("rope_dims", 8, -5), ("rope_dims", 512, -5), ("rope_dims", -16, -5), ("eps", float("nan"), -1),
                       ("rope_theta", 0.0, -1), ("rope_theta", float("inf"), -1), ("q_norm", None, -2)):
        n = fm.paged.QKNormRopeC(base, base, 1e-6, 1e4, 256)
        setattr(n, f, v)
        assert qkv(n=n) == code, (f, v)

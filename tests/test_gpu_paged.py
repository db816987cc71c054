"""GPU: the paged cache's operators against their definition in 64 bits
(paged_util).

Tolerances, from the arithmetic and before any run:
  pages, tables, counts, 4-bit codes of given rows: equal.
  norms and rotation: 32-bit arithmetic (a few 1e-7 relative to the row's
    largest value) and one rounding to bf16, half a step of 2^-8: |err| <=
    2^-8 |x| + 1e-5 max|row|.  Quantised: half a step, the rounding of the
    group's lowest value and of the scale (2^-9 each, the latter 15 times).
  attention: the weights go to bf16 once before their product with the values
    and the result goes to bf16, 2^-9 each of sum w |v|; weights and sum differ
    by the rounding of single weights, another 2^-9; doubled for 32-bit sums:
    |err| <= 2^-7 sum w |v|.  4-bit values may go to bf16 as well (2^-9 of a
    value, and through the score a similar share of the weight): 2^-6.
"""
import pytest
import torch

import paged_util as pu

pytestmark = pytest.mark.gpu


def make_batch(fm, dev, order, lens, new):
    ends = [0]
    for k in new:
        ends.append(ends[-1] + k)
    i32 = dict(dtype=torch.int32, device=dev)
    return fm.PagedBatch(torch.tensor(order, **i32), torch.tensor(ends, **i32), torch.tensor(lens, **i32), ends[-1],
                         max(new))


def check_attend(cache, q, batch, window, sinks, scale, **kw):
    got = cache.attend(0, q, batch, window, sinks, scale, **kw)
    torch.cuda.synchronize()
    want, mag = pu.attend64(cache, q, batch, window, sinks, scale)
    tol = (2.0 ** -7 if cache.bits == 16 else 2.0 ** -6) * mag
    g = got.cpu().double()
    n = batch.q_start.tolist()[-1]
    assert torch.isfinite(g[:n]).all()
    bad = (g - want)[:n].abs() - tol[:n]
    assert bad.max() <= 1e-30, (bad.max(), (g - want)[:n].abs().max())
    return got


SHAPES = [  # kv heads, heads, dim
    (8, 16, 256), (2, 16, 512), (2, 2, 256), (1, 8, 256), (2, 6, 512), (3, 15, 256),
]


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("kv_heads,heads,dim", SHAPES)
@pytest.mark.parametrize("page,lens,new,window,sinks", [
    (16, [1, 2, 15, 16, 17, 33], [1, 1, 1, 1, 1, 1], 0, 0),
    (32, [700, 31, 1, 257], [1, 1, 1, 1], 100, 4),
    (64, [130, 64, 300], [3, 64, 2], 0, 0),
    (16, [90, 200, 333], [90, 1, 37], 50, 3),
    (128, [513, 129], [130, 129], 128, 17),
    (32, [2100], [5], 1024, 4),
])
def test_attend(fm, dev, bits, kv_heads, heads, dim, page, lens, new, window, sinks):
    cache, order = pu.blank_cache(fm, dev, lens, kv_heads, dim, page, bits, seed=page + dim)
    batch = make_batch(fm, dev, order, lens, new)
    g = torch.Generator(device=dev).manual_seed(5)
    q = torch.randn(batch.tokens, heads, dim, generator=g, device=dev).bfloat16()
    a = check_attend(cache, q, batch, window, sinks, 1.5 * dim ** -0.5)
    b = cache.attend(0, q, batch, window, sinks, 1.5 * dim ** -0.5)
    assert torch.equal(a, b)  # no order of arrival in the result


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,kv_heads,heads", [(256, 8, 16), (512, 2, 16)])
def test_attend_long(fm, dev, bits, dim, kv_heads, heads):
    """Long keys with few rows (split and joined) next to short ones and a prompt."""
    lens, new = [9001, 3, 4500, 700, 1], [1, 1, 4, 700, 1]
    cache, order = pu.blank_cache(fm, dev, lens, kv_heads, dim, 32, bits, seed=1)
    batch = make_batch(fm, dev, order, lens, new)
    g = torch.Generator(device=dev).manual_seed(2)
    q = torch.randn(batch.tokens, heads, dim, generator=g, device=dev).bfloat16()
    check_attend(cache, q, batch, 0, 0, dim ** -0.5)
    check_attend(cache, q, batch, 1024, 4, dim ** -0.5)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,kv_heads,heads", [(256, 8, 16), (512, 2, 16)])
@pytest.mark.parametrize("lens,new", [
    ([9001, 3, 4500, 700, 1], [1, 1, 4, 700, 1]),
    ([700], [700]),
    ([300, 40, 900], [300, 40, 123]),
    ([64] * 60, [64] * 60),          # items of one and of two key tiles
    ([65, 129] * 40, [33, 47] * 40),
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 3)])
def test_attend_repeats(fm, dev, bits, dim, kv_heads, heads, lens, new, window, sinks):
    """Short items and items over several CTAs, again and again: the same bits, no wait given up."""
    cache, order = pu.blank_cache(fm, dev, lens, kv_heads, dim, 32, bits, seed=1)
    batch = make_batch(fm, dev, order, lens, new)
    g = torch.Generator(device=dev).manual_seed(3)
    q = torch.randn(batch.tokens, heads, dim, generator=g, device=dev).bfloat16()
    first = check_attend(cache, q, batch, window, sinks, dim ** -0.5)
    differ = sum(~torch.isfinite(o).all() | (o != first).any()
                 for o in (cache.attend(0, q, batch, window, sinks, dim ** -0.5) for _ in range(40)))
    assert int(differ) == 0
    assert cache.status() == fm.FMOE_OK


def test_attend_in_a_graph_outlives_larger_calls(fm, dev):
    """Scratch that a captured call uses is still there after a call that needed more."""
    lens = [40, 700]
    cache, order = pu.blank_cache(fm, dev, lens, 2, 256, 32, 16, seed=4)
    small, large = make_batch(fm, dev, order, lens, [1, 1]), make_batch(fm, dev, order, lens, [40, 700])
    g = torch.Generator(device=dev).manual_seed(6)
    q, ql = (torch.randn(b.tokens, 4, 256, generator=g, device=dev).bfloat16() for b in (small, large))
    stream, graph, out = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(q)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        want = cache.attend(0, q, small, scale=0.0625)
        held = cache._scratch["attend", cache._stream()]
        with torch.cuda.graph(graph, stream=stream):
            cache.attend(0, q, small, scale=0.0625, out=out)
        cache.attend(0, ql, large, scale=0.0625)
        assert any(x is held for x in list(cache._scratch.values()) + cache._outgrown)
        del held
        graph.replay()
    stream.synchronize()
    assert torch.equal(out, want)


def poison_unseen(cache, order, lens, new, window, sinks):
    """NaN and infinities in every row that no query sees."""
    seen = torch.zeros(cache.num_pages, cache.page_size, dtype=torch.bool)
    table = cache.table.cpu()
    for s, n, k in zip(order, lens, new):
        for j in range(max(0, n)):
            low = max(0, n - k - window + 1) if window else 0
            if j >= low or j < sinks:
                p = int(table[s, j // cache.page_size])
                if p >= 0:
                    seen[p, j % cache.page_size] = True
    hide = ~seen.to(cache.device)
    if cache.bits == 16:
        r = pu.rows_view(cache)[0].permute(0, 3, 1, 2, 4)          # [page, slot, ...]
        r[hide] = float("nan")
        r[..., ::7][hide] = float("inf")
    else:
        r = pu.q4_pairs(cache)[0].permute(0, 3, 1, 2, 4, 5)
        r[hide] = float("nan")


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,kv_heads,heads", [(256, 2, 4), (512, 1, 8)])
@pytest.mark.parametrize("lens,new,window,sinks", [
    ([5, 37, 300], [1, 1, 1], 0, 0),
    ([500, 900], [1, 1], 64, 4),
    ([500, 900], [100, 333], 70, 5),
    ([33, 130], [33, 130], 0, 0),
])
def test_attend_ignores_what_no_query_sees(fm, dev, bits, dim, kv_heads, heads, lens, new, window, sinks):
    cache, order = pu.blank_cache(fm, dev, lens, kv_heads, dim, 32, bits, seed=3)
    poison_unseen(cache, order, lens, new, window, sinks)
    batch = make_batch(fm, dev, order, lens, new)
    q = torch.randn(batch.tokens, heads, dim, device=dev).bfloat16()
    check_attend(cache, q, batch, window, sinks, dim ** -0.5)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_rows_that_see_nothing(fm, dev, bits, rows):
    """Sequences without positions, more new rows than positions, missing pages and ids
    outside the table: zeros, and nothing read out of bounds."""
    lens = [40, 70, 200, 64, 90]
    cache, order = pu.blank_cache(fm, dev, lens, 2, 256, 32, bits, seed=4)
    table = cache.table
    table[order[2], 1:4] = -1           # holes
    table[order[3]] = -1                # all pages gone
    table[order[4], 0] = cache.num_pages + 7
    # row 5: a table row that does not exist; rows 0, 1: no positions, fewer positions than rows
    i32 = dict(dtype=torch.int32, device=dev)
    seqs = torch.tensor(order + [cache.max_seqs + 3, -5], **i32)
    kv_len = torch.tensor([-1, 1, 200, 64, 90, 50, 20], **i32)
    q_start = torch.tensor([rows * i for i in range(8)], **i32)
    batch = fm.PagedBatch(seqs, q_start, kv_len, 7 * rows, rows)
    q = torch.randn(batch.tokens, 4, 256, device=dev).bfloat16()
    got = check_attend(cache, q, batch, 0, 0, 0.06)
    assert (got[:rows] == 0).all() and (got[rows:2 * rows - 1] == 0).all() and (got[3 * rows:4 * rows] == 0).all()
    assert (got[5 * rows:] == 0).all()
    check_attend(cache, q, batch, 16, 2, 0.06)


def test_attend_empty_batches_and_rows_past_the_end(fm, dev):
    cache, order = pu.blank_cache(fm, dev, [20], 2, 256, 16)
    empty = fm.PagedBatch(*(torch.zeros(n, dtype=torch.int32, device=dev) for n in (0, 1, 0)), 0, 0)
    assert cache.attend(0, torch.empty(0, 4, 256, device=dev, dtype=torch.bfloat16), empty).shape == (0, 4, 256)
    i32 = dict(dtype=torch.int32, device=dev)
    batch = fm.PagedBatch(torch.tensor([order[0]] * 2, **i32), torch.tensor([0, 0, 1], **i32), torch.tensor([20, 20], **i32), 3, 2)
    out = torch.full((3, 4, 256), 7.0, dtype=torch.bfloat16, device=dev)
    q = torch.randn(3, 4, 256, device=dev).bfloat16()
    cache.attend(0, q, batch, out=out)
    assert (out[1:] == 7).all() and not (out[0] == 7).all()


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("new", [1, 50])
def test_attend_strided_queries_on_another_stream(fm, dev, bits, new):
    lens = [333, 80]
    cache, order = pu.blank_cache(fm, dev, lens, 2, 256, 32, bits, seed=9)
    batch = make_batch(fm, dev, order, lens, [new, new])
    qkv = torch.randn(batch.tokens, (4 + 2 * 2) * 256 + 8, device=dev).bfloat16()
    q = qkv[:, :4 * 256].unflatten(1, (4, 256))
    assert not q.is_contiguous()
    want = check_attend(cache, q.contiguous(), batch, 0, 0, 0.06)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = cache.attend(0, q, batch, 0, 0, 0.06)
        odd = cache.attend(0, q.transpose(0, 1).contiguous().transpose(0, 1), batch, 0, 0, 0.06)  # heads apart: copied
    other.synchronize()
    assert torch.equal(got, want) and torch.equal(odd, want)


def test_attend_pages_past_4_gb(fm, dev):
    """Pages whose byte offset passes 32 bits."""
    cache = fm.PagedKVCache(1, 8, 256, 4600, 2, 4, 128, device=dev)
    ids = [4599, 2, 4301, 4200]
    cache.table[0] = torch.tensor(ids, dtype=torch.int32, device=dev)
    cache.refs[ids] = 1
    for layer_page in ids:
        pu.rows_view(cache)[0, layer_page] = torch.randn(8, 2, 128, 256, device=dev)
    lens, new = [512], [130]
    batch = make_batch(fm, dev, [0], lens, new)
    k, v = (torch.randn(130, 8, 256, device=dev).bfloat16() for _ in range(2))
    cache.append(0, k, v, batch)
    pos = torch.arange(382, 512)
    page = torch.tensor(ids)[pos // 128]
    assert torch.equal(pu.rows_view(cache)[0, page, :, 0, pos % 128], k)
    q = torch.randn(130, 16, 256, device=dev).bfloat16()
    got = cache.attend(0, q, batch, 0, 0, 0.06)
    k_all, v_all = (pu.rows_view(cache)[0, torch.tensor(ids), :, i].transpose(1, 2).reshape(512, 8, 256).double()
                    .repeat_interleave(2, 1) for i in (0, 1))
    s = torch.einsum("qhd,nhd->hqn", q.double(), k_all) * 0.06
    s = s.masked_fill(torch.arange(512, device=dev) > pos.to(dev)[:, None], float("-inf"))
    w = torch.softmax(s, -1)
    err = (got.double() - torch.einsum("hqn,nhd->qhd", w, v_all)).abs()
    assert (err <= 2.0 ** -7 * torch.einsum("hqn,nhd->qhd", w, v_all.abs())).all()


@pytest.mark.parametrize("scale", [40.0, -1.0, 0.0])
@pytest.mark.parametrize("new", [1, 33])
def test_attend_large_scores(fm, dev, scale, new):
    """One weight near 1 (scores in the thousands), scores of either sign, all equal.
    A score's 32-bit error (2^-22 of the sum of its terms' magnitudes) moves a
    weight by as much: at scale 40 a few 1e-3, inside the tolerance's slack."""
    cache, order = pu.blank_cache(fm, dev, [600, 70], 2, 256, 32, seed=6)
    batch = make_batch(fm, dev, order, [600, 70], [new, new])
    q = torch.randn(batch.tokens, 4, 256, device=dev).bfloat16()
    check_attend(cache, q, batch, 0, 0, scale)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("dim,kv_heads,heads", [(256, 2, 4), (512, 1, 8)])
@pytest.mark.parametrize("size,q_size", [(1500.0, 2.0 ** -60), (2.0 ** -9, 2.0 ** 60), (1.0, 0.0)])
def test_attend_4bit_values_and_queries_of_any_size(fm, dev, new, dim, kv_heads, heads, size, q_size):
    """Scales from 2^-9 to 1500 (values to 12000), queries from 2^-60 to 2^60, zeros.
    Scores of a deviation of 1/2: with values to 2^-12 (three times that for a whole
    group) a weight is off by 2^-11 of the sum of its score's magnitudes, about 6."""
    lens = [700, 90]
    cache, order = pu.blank_cache(fm, dev, lens, kv_heads, dim, 32, 4, seed=9)
    pairs = pu.q4_pairs(cache)
    g = torch.Generator(device=dev).manual_seed(7)
    s = size * (0.5 + 0.5 * torch.rand(pairs.shape[:-1], generator=g, device=dev))
    pairs[..., 0] = s.bfloat16()
    pairs[..., 1] = (-7.5 * s).bfloat16()
    batch = make_batch(fm, dev, order, lens, [new, new])
    q = (q_size * torch.randn(batch.tokens, heads, dim, generator=g, device=dev)).bfloat16()
    q[0, 0] = 0
    scale = 0.5 / (dim ** 0.5 * 4.6 * 0.75 * size * q_size) if q_size else 1.0
    check_attend(cache, q, batch, 0, 0, scale)
    check_attend(cache, q, batch, 64, 3, scale)


# ---- rows ------------------------------------------------------------------------


def quantise32(x):
    """fp32 rows [..., D] -> (codes, scale, bias) as fmoe_quantize defines them."""
    g = x.float().unflatten(-1, (-1, 64))
    mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((mx - mn) / 15).clamp(min=1e-7).bfloat16()
    b = mn.bfloat16()
    return torch.round((g - b.float()) / s.float()).clamp(0, 15).flatten(-2).long(), s.squeeze(-1), b.squeeze(-1)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,page", [(256, 16), (512, 64)])
def test_append_stores_rows_as_they_are(fm, dev, bits, dim, page):
    lens, new = [70, 5, 129, 33], [70, 1, 30, 0]
    cache, order = pu.blank_cache(fm, dev, lens, 3, dim, page, bits, layers=2, seed=8)
    before = cache.pages.clone()
    batch = make_batch(fm, dev, order, lens, new)
    kv = torch.randn(batch.tokens, 2 * 3 * dim, device=dev).bfloat16()
    kv[3] = 0.0  # a row without a range
    k, v = kv[:, :3 * dim].unflatten(1, (3, dim)), kv[:, 3 * dim:].unflatten(1, (3, dim))
    cache.append(1, k, v, batch)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
    seq = torch.cat([torch.full((m,), s) for s, m in zip(order, new)])
    p, s = cache.table.cpu()[seq, pos // page].long().to(dev), (pos % page).to(dev)
    rows = torch.stack([k, v], 2)
    if bits == 16:
        assert torch.equal(pu.rows_view(cache)[1, p, :, :, s], rows)
        old = before.view(torch.bfloat16).view_as(pu.rows_view(cache)).clone()
        old[1, p, :, :, s] = rows
        assert torch.equal(old, pu.rows_view(cache))  # nothing else changed
    else:
        codes, sc, bi = quantise32(rows)
        assert torch.equal(pu.q4_codes(cache)[1, p, :, :, s], codes)
        assert torch.equal(pu.q4_pairs(cache)[1, p, :, :, s], torch.stack([sc, bi], -1))
        changed = (pu.blocks_view(cache) != before.view_as(pu.blocks_view(cache))).flatten(2).any(-1)
        assert not changed[0].any() and set(changed[1].nonzero()[:, 0].tolist()) <= set(p.tolist())


def turned64(x, w, pos, rope, theta, eps=1e-6):
    x = x.cpu().double()
    x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    if w is None:
        return x
    x = x * w.cpu().double()
    h = rope // 2
    ang = pos.double()[:, None, None] * theta ** (-torch.arange(h).double() / max(h, 1))
    a, b = x[..., :h], x[..., h:2 * h]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., 2 * h:]], -1)


@pytest.mark.parametrize("bits", [16, 4])
@pytest.mark.parametrize("dim,heads,kv_heads,rope,theta,shared", [
    (256, 16, 8, 256, 1e4, False), (512, 16, 2, 128, 1e6, True), (256, 3, 1, 16, 1e4, False), (512, 5, 1, 512, 1e6, False),
    (256, 2, 2, 0, 1e4, False),
])
def test_append_qkv(fm, dev, bits, dim, heads, kv_heads, rope, theta, shared):
    lens, new = [300000, 40, 17, 129], [3, 40, 1, 60]
    page = 128
    # the far sequence holds only its last pages
    cache = fm.PagedKVCache(1, kv_heads, dim, 16, 4, 300000 // page + 2, page, bits, device=dev)
    nxt = iter(range(16))
    for i, (n, m) in enumerate(zip(lens, new)):
        for b in range((n - m) // page, -(-n // page)):
            cache.table[i, b] = next(nxt)
    batch = make_batch(fm, dev, [0, 1, 2, 3], lens, new)
    T = batch.tokens
    x = (torch.randn(T, (heads + 2 * kv_heads) * dim, device=dev) * 3).bfloat16()
    q, k, v = (t.unflatten(1, (-1, dim)) for t in x.split([heads * dim, kv_heads * dim, kv_heads * dim], 1))
    qn, kn = ((1 + 0.3 * torch.randn(dim, device=dev)).bfloat16() for _ in range(2))
    got = cache.append_qkv(0, q, k, None if shared else v, batch, fm.QKNormRope(qn, kn, rope, theta))
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)])
    seq = torch.cat([torch.full((m,), i) for i, m in enumerate(new)])
    want_q, want_k = turned64(q, qn, pos, rope, theta), turned64(k, kn, pos, rope, theta)
    want_v = turned64(k if shared else v, None, pos, 0, theta)
    close = lambda a, b: ((a.cpu().double() - b).abs() <= 2.0 ** -8 * b.abs() + 1e-5 * b.abs().amax(-1, keepdim=True)).all()  # noqa: E731
    assert close(got, want_q)
    p, s = cache.table.cpu()[seq, pos // page].long(), pos % page
    stored = pu.values(cache)[p, :, :, s]                                        # [T, kv heads, 2, dim]
    for i, want in ((0, want_k), (1, want_v)):
        if bits == 16:
            assert close(stored[:, :, i], want)
            continue
        g = want.unflatten(-1, (-1, 64))
        mn, mx = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
        step = (mx - mn) / 15
        tol = 0.5 * step * (1 + 2.0 ** -8) + 2.0 ** -9 * (mn.abs() + 15 * step) + 1e-5 * g.abs().amax(-1, keepdim=True)
        assert ((stored[:, :, i].unflatten(-1, (-1, 64)) - g).abs() <= tol).all()


def test_append_drops_positions_without_a_page(fm, dev):
    cache, order = pu.blank_cache(fm, dev, [64, 20], 1, 256, 16, seed=2)
    cache.table[order[0], 1] = -1
    before = pu.rows_view(cache).clone()
    i32 = dict(dtype=torch.int32, device=dev)
    batch = fm.PagedBatch(torch.tensor(order + [99], **i32), torch.tensor([0, 64, 74, 80], **i32),
                          torch.tensor([64, -1, 6], **i32), 80, 64)
    k = torch.randn(80, 1, 256, device=dev).bfloat16()
    cache.append(0, k, k, batch)
    after = pu.rows_view(cache)
    kept = torch.tensor([j for j in range(64) if j // 16 != 1])
    p = cache.table.cpu()[order[0], kept // 16].long()
    assert torch.equal(after[0, p, :, 0, kept % 16].cpu(), k[kept.to(dev)].cpu())
    before[0, p, :, :, kept % 16] = after[0, p, :, :, kept % 16]
    assert torch.equal(before, after)


# ---- pages -----------------------------------------------------------------------


@pytest.mark.parametrize("bits,dim,page,layers", [(16, 256, 16, 3), (4, 512, 32, 2), (4, 256, 128, 1)])
def test_pages_follow_the_host_model(fm, dev, bits, dim, page, layers):
    """A long random life of a small pool: tables, lengths, counts, what every live page
    holds and the refusals are those of the host model after each call."""
    import random

    r = random.Random(page)
    cache = fm.PagedKVCache(layers, 2, dim, 37, 9, 6, page, bits, device=dev)
    cache.pages.zero_()
    host = pu.HostPages(cache)
    stamp = 0
    flat = cache.pages.view(torch.uint8).view(layers, 37, -1)
    for step in range(120):
        op = r.choice(["reserve"] * 4 + ["fork"] * 3 + ["free", "trim", "compact"])
        if op == "reserve":
            seqs = r.sample(range(9), r.randint(1, 9))
            new = [r.choice([0, 1, 1, page - 1, page, 2 * page + 3, 7 * page]) for _ in seqs]
            batch = cache.reserve(seqs, new)
            want = host.reserve(seqs, new)
            assert batch.kv_len.tolist() == want and batch.tokens == sum(new)
            for s in seqs:  # mark the sequence's own pages with what they hold
                for p in host.table[s]:
                    if p >= 0 and host.refs[p] == 1:
                        stamp += 1
                        host.content[p] = stamp % 251
                        flat[:, p] = stamp % 251
        elif op == "fork":
            rows = r.sample(range(9), 9)
            k = r.randint(1, 6)
            parents = [r.choice(rows[k:]) for _ in range(k)]
            cache.fork(parents, rows[:k])
            host.fork(parents, rows[:k])
        elif op == "free":
            seqs = r.sample(range(9), r.randint(1, 3))
            cache.free(seqs)
            host.free(seqs)
        elif op == "trim":
            seqs, w, s = r.sample(range(9), 4), r.choice([1, 5, page + 1]), r.choice([0, 3, page])
            cache.trim(seqs, w, s)
            host.trim(seqs, w, s)
        else:
            assert cache.compact().item() == host.compact()
        assert cache.table.tolist() == host.table and cache.lens.tolist() == host.lens, (step, op)
        assert cache.refs.tolist() == host.refs and cache.refused.item() == host.refused, (step, op)
        live = [p for p in range(37) if host.refs[p] and host.content[p] is not None]
        want = torch.tensor([host.content[p] for p in live], dtype=torch.uint8, device=dev)
        assert (flat[:, live] == want[None, :, None]).all(), (step, op)
    assert host.refused > 0 and max(host.refs) > 1


def test_reserve_many_sequences(fm, dev):
    """More sequences than the planning CTA has threads, and a pool that runs out on the way."""
    cache = fm.PagedKVCache(1, 1, 256, 3000, 2500, 3, 16, 4, device=dev)
    host = pu.HostPages(cache)
    g = torch.Generator().manual_seed(1)
    seqs = torch.randperm(2500, generator=g).tolist()
    for most in (20, 30, 60):
        new = torch.randint(0, most, (2500,), generator=g).tolist()
        batch = cache.reserve(seqs, new)
        assert batch.kv_len.tolist() == host.reserve(seqs, new)
        assert cache.table.tolist() == host.table and cache.refs.tolist() == host.refs
        assert cache.refused.item() == host.refused
    assert host.refused > 0


def test_fork_refuses_crossed_pairs_on_the_device(fm, dev):
    cache, order = pu.blank_cache(fm, dev, [20, 40], 1, 256, 16, rows=6, spare=6)
    a, b = order
    c, d = [s for s in range(6) if s not in order][:2]
    i32 = dict(dtype=torch.int32, device=dev)
    table = cache.table.clone()
    # (a -> c) stands; (b -> c) names c again; (c -> a) makes a parent a child; ids outside the table
    cache.fork(torch.tensor([a, b, b, 77, -1], **i32), torch.tensor([c, c, a, d, 6], **i32))
    assert cache.refused.item() == 4
    assert torch.equal(cache.table[[a, b, d]], table[[a, b, d]])
    assert cache.lens[c] == 20 and cache.table[c, 0] == table[a, 0] and cache.table[c, 1] != table[a, 1]


def test_copy_pages(fm, dev):
    cache, _ = pu.blank_cache(fm, dev, [64], 2, 512, 16, 4, layers=3, spare=20, seed=5)
    want = pu.blocks_view(cache).clone()
    src, dst = [1, 1, 9, 4], [2, 3, 10, 0]
    want[:, dst] = want[:, src]
    cache.copy_pages(src, dst)
    assert torch.equal(pu.blocks_view(cache), want)


def test_a_captured_decode_loop_grows_its_sequences(fm, dev):
    """reserve, append_qkv and attend in one CUDA graph: each replay adds a position."""
    cache = fm.PagedKVCache(1, 2, 256, 40, 3, 8, 16, device=dev)
    i32 = dict(dtype=torch.int32, device=dev)
    seqs, one = torch.tensor([2, 0], **i32), torch.ones(2, **i32)
    norm = fm.QKNormRope(torch.ones(256, device=dev), torch.ones(256, device=dev), 256, 1e4)
    x = torch.randn(2, 8, 256, device=dev).bfloat16()

    def step():
        batch = cache.reserve(seqs, one, tokens=2, max_new=1)
        q = cache.append_qkv(0, x[:, :4], x[:, 4:6], x[:, 6:], batch, norm)
        return batch, q, cache.attend(0, q, batch, window=20, sinks=2, scale=0.06)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()  # scratch exists before the capture
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            batch, q, out = step()
    torch.cuda.synchronize()
    for n in range(2, 60):
        x.copy_(torch.randn(2, 8, 256, device=dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert batch.kv_len.tolist() == [n, n] and cache.lens.tolist() == [n, 0, n]
        want, mag = pu.attend64(cache, q, batch, 20, 2, 0.06)
        assert ((out.cpu().double() - want).abs() <= 2.0 ** -7 * mag).all(), n


# ---- refusals --------------------------------------------------------------------


def test_python_refusals(fm, dev):
    cache, order = pu.blank_cache(fm, dev, [40, 40], 2, 256, 16)
    batch = make_batch(fm, dev, order, [40, 40], [1, 1])
    q = torch.zeros(2, 4, 256, dtype=torch.bfloat16, device=dev)
    for bad in (lambda: cache.attend(0, q.cpu(), batch), lambda: cache.attend(0, q[:1], batch),
                lambda: cache.attend(0, q[..., :128], batch), lambda: cache.append(0, q, q, batch),
                lambda: cache.attend(0, q, batch, out=torch.empty(2, 4, 256, device=dev)),
                lambda: cache.reserve([0, 0], [1, 1]), lambda: cache.reserve([0], [1, 1]),
                lambda: cache.reserve([0], [-1]), lambda: cache.fork([0], [0]), lambda: cache.fork([0, 1], [2, 2]),
                lambda: cache.free([1, 1]), lambda: cache.copy_pages([0, 1], [1, 2]),
                lambda: cache.free(torch.zeros(1, dtype=torch.int64, device=dev)),
                lambda: cache.reserve(torch.zeros(1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)),
                lambda: fm.PagedBatch(batch.seqs, batch.seqs, batch.kv_len, 2, 1),
                lambda: fm.PagedBatch(batch.seqs, batch.q_start, batch.kv_len, 3, 1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: cache.attend(1, q, batch), lambda: cache.attend(0, q[:, :3], batch),
                lambda: cache.attend(0, q, batch, window=-1), lambda: cache.attend(0, q, batch, sinks=-1),
                lambda: cache.attend(0, q, batch, scale=float("nan")), lambda: cache.trim([0], 0),
                lambda: cache.attend(0, torch.zeros(2, 18, 256, dtype=torch.bfloat16, device=dev), batch),
                lambda: cache.append_qkv(0, q, q[:, :2], None, batch, fm.QKNormRope(q[0, 0], q[0, 0], 8, 1e4)),
                lambda: cache.append_qkv(0, q, q[:, :2], None, batch, fm.QKNormRope(q[0, 0], q[0, 0], 256, 0.0)),
                lambda: fm.PagedKVCache(1, 2, 128, 4, 1, 1), lambda: fm.PagedKVCache(1, 2, 256, 4, 1, 1, 24),
                lambda: fm.PagedKVCache(1, 2, 256, 4, 1, 1, 16, 8), lambda: fm.PagedKVCache(0, 2, 256, 4, 1, 1)):
        with pytest.raises(fm.FmoeError):
            bad()

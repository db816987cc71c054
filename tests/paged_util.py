"""The paged cache in plain 64-bit form: what the pages hold, the attention over
them, and a host model of who holds which page."""
import torch


def blank_cache(fm, dev, lens, kv_heads, dim, page, bits=16, layers=1, spare=3, seed=0, rows=None, fill=True):
    """A cache whose sequence i (table row order[i]) holds lens[i] positions in pages
    of random ids, with random rows; returns (cache, rows of the table)."""
    g = torch.Generator().manual_seed(seed)
    blocks = [-(-n // page) for n in lens]
    count = sum(blocks) + spare
    rows = rows or len(lens) + 2
    cache = fm.PagedKVCache(layers, kv_heads, dim, count, rows, max(blocks, default=0) + 2, page, bits, device=dev)
    ids = torch.randperm(count, generator=g).tolist()
    order = torch.randperm(rows, generator=g).tolist()[: len(lens)]
    table, refs, held = cache.table.cpu(), cache.refs.cpu(), cache.lens.cpu()
    for i, nb in enumerate(blocks):
        for b in range(nb):
            table[order[i], b] = p = ids.pop()
            refs[p] = 1
        held[order[i]] = lens[i]
    cache.table.copy_(table)
    cache.refs.copy_(refs)
    cache.lens.copy_(held)
    if fill:
        gd = torch.Generator(device=dev).manual_seed(seed + 1)
        if bits == 16:
            cache.pages.view(torch.bfloat16).copy_(torch.randn(cache.pages.numel() // 2, generator=gd, device=dev))
        else:
            raw = torch.randint(0, 256, (cache.pages.numel(),), generator=gd, device=dev, dtype=torch.uint8)
            cache.pages.copy_(raw)
            pairs = q4_pairs(cache)
            s = torch.rand(pairs.shape[:-1], generator=gd, device=dev) * 0.2 + 0.1
            pairs[..., 0] = s
            pairs[..., 1] = -7.5 * s + 0.1 * torch.randn(s.shape, generator=gd, device=dev)
    return cache, order


def blocks_view(cache):
    return cache.pages.view(torch.uint8).view(cache.layers, cache.num_pages, cache.kv_heads, 2, -1)


def rows_view(cache):
    """bf16 rows [layers, pages, kv heads, 2, page_size, dim]."""
    return cache.pages.view(torch.bfloat16).view(cache.layers, cache.num_pages, cache.kv_heads, 2, cache.page_size,
                                                 cache.head_dim)


def q4_pairs(cache):
    """(scale, bias) [layers, pages, kv heads, 2, page_size, dim / 64, 2], a view."""
    at = cache.page_size * cache.head_dim // 2
    return blocks_view(cache).view(torch.bfloat16)[..., at // 2:].unflatten(-1, (cache.page_size, cache.head_dim // 64, 2))


def q4_codes(cache):
    """Codes [layers, pages, kv heads, 2, page_size, dim], natural order of values."""
    D, at = cache.head_dim, cache.page_size * cache.head_dim // 2
    w = blocks_view(cache)[..., :at].contiguous().view(torch.int32).unflatten(-1, (cache.page_size, D // 8)).long()
    d = torch.arange(D, device=w.device)
    word = (d % 64 // 8) * (D // 64) + d // 64
    return (w[..., word] >> (4 * (d % 8 // 2 + 4 * (d % 2)))) & 15


def values(cache, layer=0):
    """Every row as 64-bit values [pages, kv heads, 2, page_size, dim] on the CPU."""
    if cache.bits == 16:
        return rows_view(cache)[layer].cpu().double()
    p = q4_pairs(cache)[layer].cpu().double().repeat_interleave(64, dim=-2)
    return q4_codes(cache)[layer].cpu().double() * p[..., 0] + p[..., 1]


def attend64(cache, q, batch, window, sinks, scale, layer=0):
    """(attention, sum of weights times |values|) of every row, in 64 bits."""
    vals, table = values(cache, layer), cache.table.cpu()
    q = q.cpu().double()
    starts, lens, seqs = batch.q_start.tolist(), batch.kv_len.tolist(), batch.seqs.tolist()
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    share = q.shape[1] // cache.kv_heads
    for b, n in enumerate(lens):
        a, z = starts[b], starts[b + 1]
        if n <= 0 or z == a:
            continue
        j = torch.arange(n)
        page = table[seqs[b]][j // cache.page_size].long() if 0 <= seqs[b] < cache.max_seqs else torch.full((n,), -1)
        held = (page >= 0) & (page < cache.num_pages)
        kv = vals[page.clamp(0, cache.num_pages - 1), :, :, j % cache.page_size]      # [n, kv heads, 2, dim]
        p = torch.arange(a, z) + n - z
        see = held & (j <= p[:, None])
        if window:
            see &= (j > p[:, None] - window) | (j < sinks)
        seen = see.any(0)
        kv = torch.where(seen[:, None, None, None], kv, 0.0)
        k, v = (kv[:, :, i].repeat_interleave(share, 1) for i in (0, 1))
        s = torch.einsum("qhd,nhd->hqn", q[a:z], k) * scale
        s = s.masked_fill(~see, float("-inf"))
        w = torch.softmax(s, -1).nan_to_num(0.0)
        out[a:z] = torch.einsum("hqn,nhd->qhd", w, v)
        mag[a:z] = torch.einsum("hqn,nhd->qhd", w, v.abs())
    return out, mag


class HostPages:
    """Who holds which page, and what each page holds (a number for each layer)."""

    def __init__(self, cache):
        self.page, self.blocks, self.n = cache.page_size, cache.max_blocks, cache.num_pages
        self.table = [[-1] * cache.max_blocks for _ in range(cache.max_seqs)]
        self.lens, self.refs = [0] * cache.max_seqs, [0] * cache.num_pages
        self.content = [None] * cache.num_pages
        self.refused = 0

    def _free(self):
        return [p for p, n in enumerate(self.refs) if n == 0]

    def _count(self, n):
        return -(-n // self.page)

    def reserve(self, seqs, new):
        free, got, used = self._free(), [], 0
        for s, k in zip(seqs, new):
            have = self._count(self.lens[s])
            need = self._count(self.lens[s] + k) - have
            if self.lens[s] + k > self.blocks * self.page:
                got.append(-1)
                self.refused += 1
                continue
            used += need
            if need and used > len(free):
                got.append(-1)
                self.refused += 1
                continue
            for i in range(need):
                p = free[used - need + i]
                self.table[s][have + i] = p
                self.refs[p] = 1
            self.lens[s] += k
            got.append(self.lens[s])
        return got

    def _release(self, s, blocks):
        for b in blocks:
            p = self.table[s][b]
            if p >= 0:
                self.refs[p] -= 1
                self.table[s][b] = -1

    def free(self, seqs):
        for s in seqs:
            self._release(s, range(self.blocks))
            self.lens[s] = 0

    def trim(self, seqs, window, sinks):
        for s in seqs:
            self._release(s, [b for b in range(self.blocks)
                              if b * self.page >= sinks and (b + 1) * self.page <= self.lens[s] - window + 1])

    def fork(self, parents, children):
        for d in children:
            self._release(d, range(self.blocks))
            self.lens[d] = 0
        free, k = self._free(), 0
        for a, d in zip(parents, children):
            part = self.lens[a] % self.page and self.table[a][self.lens[a] // self.page] >= 0
            if part:
                k += 1
                if k > len(free):
                    self.refused += 1
                    continue
            self.table[d] = list(self.table[a])
            self.lens[d] = self.lens[a]
            if part:
                b = self.lens[a] // self.page
                self.table[d][b] = free[k - 1]
                self.content[free[k - 1]] = self.content[self.table[a][b]]
            for p in self.table[d]:
                if p >= 0:
                    self.refs[p] += 1

    def compact(self):
        n = sum(1 for r in self.refs if r)
        src = [p for p in range(n, self.n) if self.refs[p]]
        dst = [p for p in range(n) if not self.refs[p]]
        to = dict(zip(src, dst))
        for s, d in to.items():
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.content[d] = self.content[s]
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return n

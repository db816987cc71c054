"""Measured cases of the paged KV cache's operators: attention with a sliding window and visible first tokens over
bf16 pages and over 4-bit pages, the pass that norms, rotates and stores new rows, and forking and compacting pages.

    listed()             the cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  a server's state before the call: pages, block table, new rows
    run(state)           one call, in plain tensor operations or (own) through the package
    work(case)           bytes and operations that the call cannot do without
    exact(case, seed)    the same answer in 64 bits, from the definition

Pages are [layer][page][kv head][K | V][rows]; a bf16 row is head_dim values, a 4-bit row head_dim / 8 words of
codes, and behind the codes of a page's rows one bf16 (scale, bias) pair for each 64 values of each row.  The word
of octet o of group g lies at o * (head_dim / 64) + g; value i of an octet is nibble (i >> 1) + 4 * (i & 1).
"""
import random

import torch

own = False

SLIDING = {"heads": 16, "kv_heads": 8, "dim": 256}  # the two attention shapes of the package's Gemma-4 configuration
FULL = {"heads": 16, "kv_heads": 2, "dim": 512}


def listed():
    return [
        # one user, early in a chat: a sliding layer's step, where latency counts
        {"name": "decode 1 short", "op": "attend", **SLIDING, "bits": 16, "page": 32, "seqs": 1, "least": 201, "most": 201, "new": 1,
         "mixed": False, "window": 1024, "sinks": 4},
        # a full batch on a full-attention layer, lengths from a greeting to a long document
        {"name": "decode 32 ragged", "op": "attend", **FULL, "bits": 16, "page": 32, "seqs": 32, "least": 17, "most": 16001, "new": 1,
         "mixed": False, "window": 0, "sinks": 0},
        # a large batch of long chats on a sliding layer whose pages out of the window are freed
        {"name": "decode 64 window sinks", "op": "attend", **SLIDING, "bits": 16, "page": 16, "seqs": 64, "least": 500, "most": 32768,
         "new": 1, "mixed": False, "window": 1024, "sinks": 4},
        # one prompt on a sliding layer
        {"name": "prompt 4096 window sinks", "op": "attend", **SLIDING, "bits": 16, "page": 64, "seqs": 1, "least": 4096, "most": 4096,
         "new": 4096, "mixed": False, "window": 1024, "sinks": 4},
        # a step that mixes chunks of prompts with running decodes, on a full-attention layer
        {"name": "chunks and decodes", "op": "attend", **FULL, "bits": 16, "page": 32, "seqs": 12, "least": 601, "most": 6007, "new": 385,
         "mixed": True, "window": 0, "sinks": 0},
        # a few users over 4-bit pages
        {"name": "4-bit decode 4", "op": "attend", **SLIDING, "bits": 4, "page": 32, "seqs": 4, "least": 100, "most": 1500, "new": 1,
         "mixed": False, "window": 0, "sinks": 0},
        # the memory-bound batch that 4-bit pages are for
        {"name": "4-bit decode 48 long", "op": "attend", **SLIDING, "bits": 4, "page": 32, "seqs": 48, "least": 1000, "most": 16384,
         "new": 1, "mixed": False, "window": 0, "sinks": 0},
        # chunks of two long prompts over 4-bit pages
        {"name": "4-bit chunk 1024", "op": "attend", **SLIDING, "bits": 4, "page": 64, "seqs": 2, "least": 4100, "most": 8192, "new": 1024,
         "mixed": False, "window": 0, "sinks": 0},
        # a decode step's projections on a full-attention layer (values are the raw keys, a quarter of the dims turn)
        {"name": "rows of 24 decodes", "op": "append", **FULL, "page": 32, "seqs": 24, "least": 30, "most": 9000, "new": 1, "rope": 128,
         "theta": 1e6, "shared": True},
        # three prompts' projections on a sliding layer
        {"name": "rows of 3 prompts", "op": "append", **SLIDING, "page": 16, "seqs": 3, "least": 1501, "most": 2499, "new": 2048,
         "rope": 256, "theta": 1e4, "shared": False},
        # several answers sampled from each prompt: children share full pages and copy the part-filled one, in 25 sliding layers
        {"name": "fork 6 into 48", "op": "fork", **SLIDING, "page": 16, "layers": 25, "parents": 6, "children": 48, "least": 200,
         "most": 1000, "spare": 64},
        # a half-empty pool of 5 full-attention layers brought together before it shrinks
        {"name": "compact 2048 pages", "op": "compact", **FULL, "page": 32, "layers": 5, "pages": 2048, "live": 50, "seqs": 16},
    ]


LARGEST = 2.2e9, 3.2e11  # bytes and operations that a drawn case stays under: the listed cases' most


def _log(rng, least, most):
    return min(most, max(least, round(least * (most / least) ** rng.random())))


def draw(rng):
    while True:
        dim = rng.choice((256, 256, 512))
        kv_heads = rng.choice((2, 4, 8) if dim == 256 else (2, 2, 4))
        shape = {"heads": kv_heads * rng.choice((1, 2, 4, 8)), "kv_heads": kv_heads, "dim": dim}
        page = rng.choice((16, 32, 64))
        op = rng.choice(("attend", "attend", "attend", "append", "fork", "compact"))
        most = _log(rng, 60, 16384)
        lengths = {"least": max(1, round(most * rng.uniform(0.05, 1.0))), "most": most}
        if op == "attend":
            new = 1 if rng.random() < 0.5 else _log(rng, 2, 2048)
            case = {"op": op, **shape, "bits": rng.choice((16, 4)), "page": page, "seqs": _log(rng, 1, 64 if new == 1 else 8), **lengths,
                    "new": new, "mixed": new > 1 and rng.random() < 0.3, "window": rng.choice((0, 0, 1024, _log(rng, 100, 4096))), "sinks": 0}
            case["sinks"] = rng.choice((0, 4, 4, 17)) if case["window"] else 0
        elif op == "append":
            shared = rng.random() < 0.3
            case = {"op": op, **shape, "page": page, "seqs": _log(rng, 1, 64), **lengths, "new": rng.choice((1, _log(rng, 2, 2048))),
                    "rope": rng.choice((dim, dim // 4)), "theta": rng.choice((1e4, 1e6)), "shared": shared}
        elif op == "fork":
            parents = _log(rng, 1, 16)
            case = {"op": op, **shape, "page": page, "layers": rng.choice((1, 5, 25)), "parents": parents,
                    "children": parents * _log(rng, 1, 12), "least": max(1, most // 16), "most": max(1, most // 8), "spare": _log(rng, 8, 256)}
        else:
            case = {"op": op, **shape, "page": page, "layers": rng.choice((1, 5)), "pages": _log(rng, 64, 2048), "live": rng.randint(20, 90),
                    "seqs": _log(rng, 1, 32)}
        w = work(case)
        pool = _pool_bytes(case)
        if w["bytes"] <= LARGEST[0] and w["flops"] <= LARGEST[1] and pool <= 4e9 and _plain_values(case) <= 4e9:
            return case


# ---- what a case says, in whole numbers ---------------------------------------------------------------------------


def _lengths(case):
    """Length of every sequence: spread over the logarithm, in a fixed order of no pattern."""
    n = case.get("seqs") or case["parents"]
    a, b = case["least"], case["most"]
    got = [round(a * (b / a) ** (i / max(1, n - 1))) for i in range(n)] if n > 1 else [b]
    random.Random(n).shuffle(got)
    return got


def _new(case):
    return [1 if case.get("mixed") and i % 2 else min(case["new"], n) for i, n in enumerate(_lengths(case))]


def _visible(case):
    """For every sequence: (visible pairs of a query and a key, keys that some query sees)."""
    for n, new in zip(_lengths(case), _new(case)):
        w, s = case["window"], case["sinks"]
        if not w:
            yield sum(range(n - new + 1, n + 1)), n
            continue
        pairs = sum(min(p + 1, w) + max(0, min(s, p + 1 - w)) for p in range(n - new, n))
        low = max(0, n - new - w + 1)
        yield pairs, n - low + min(s, low)


def _row_bytes(case):
    return 2 * case["dim"] if case.get("bits", 16) == 16 else case["dim"] // 2 + case["dim"] // 16


def _page_bytes(case):
    return case["kv_heads"] * 2 * case["page"] * _row_bytes(case)


def _blocks(n, case):
    return -(-n // case["page"])


def _seen(n, new, case):
    """Blocks of a sequence that hold a page: all, or those that its window and first tokens reach."""
    w, low = case.get("window", 0), max(0, n - new - case.get("window", 0) + 1)
    return [b for b in range(_blocks(n, case)) if not w or (b + 1) * case["page"] > low or b * case["page"] < case["sinks"]]


def _pool_bytes(case):
    if case["op"] == "compact":
        return case["pages"] * case["layers"] * _page_bytes(case)
    if case["op"] == "fork":
        return (sum(_blocks(n, case) for n in _lengths(case)) + case["children"] + case["spare"]) * case["layers"] * _page_bytes(case)
    return sum(len(_seen(n, new, case)) for n, new in zip(_lengths(case), _new(case))) * _page_bytes(case)


def _plain_values(case):
    """Values of the largest padded tensor that the plain form makes."""
    if case["op"] != "attend":
        return 0
    keys = _span(case)
    return case["seqs"] * keys * max(2 * case["kv_heads"] * case["dim"], case["heads"] * max(_new(case)))


def _span(case):
    """Key positions that the plain form looks at for each sequence."""
    n, new = max(_lengths(case)), max(_new(case))
    return min(n, case["sinks"] + case["window"] + new - 1) if case["window"] else n


def work(case):
    if case["op"] == "attend":
        seen = list(_visible(case))
        rows, pairs, tokens = sum(k for _, k in seen), sum(p for p, _ in seen), sum(_new(case))
        kv = rows * case["kv_heads"] * 2 * _row_bytes(case)
        return {"bytes": kv + 4 * tokens * case["heads"] * case["dim"], "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "append":
        tokens, kv = sum(_new(case)), case["kv_heads"]
        rows = case["heads"] + (1 if case["shared"] else 2) * kv + case["heads"] + 2 * kv
        return {"bytes": 2 * case["dim"] * tokens * rows, "flops": 10 * case["dim"] * tokens * (case["heads"] + 2 * kv)}
    if case["op"] == "fork":
        lens = _lengths(case)
        copied = sum(1 for i in range(case["children"]) if lens[i % len(lens)] % case["page"])
        entries = sum(_blocks(lens[i % len(lens)], case) for i in range(case["children"]))
        return {"bytes": 2 * copied * case["layers"] * _page_bytes(case) + 8 * entries, "flops": 0}
    moved = _moves(case)
    return {"bytes": 2 * moved * case["layers"] * _page_bytes(case) + 16 * case["pages"], "flops": 0}


def _live(case):
    """Which pages of a pool to compact are live: the same for every seed, so that the work is known."""
    ids = list(range(case["pages"]))
    random.Random(case["pages"]).shuffle(ids)
    return sorted(ids[: max(1, case["pages"] * case["live"] // 100)])


def _moves(case):
    live = _live(case)
    return sum(1 for p in live if p >= len(live))


# ---- inputs --------------------------------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _quantised(x):
    """Rows [..., dim] as 4-bit codes (bytes) and (scale, bias) pairs."""
    dim = x.shape[-1]
    g = x.unflatten(-1, (dim // 64, 64))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    scale = ((high - low) / 15).clamp(min=1e-7).bfloat16()
    bias = low.bfloat16()
    code = torch.round((g - bias.float()) / scale.float()).clamp(0, 15).to(torch.uint8)
    code = code.unflatten(-1, (8, 8)).transpose(-3, -2)                       # [..., octet, group, 8]
    code = code[..., [0, 2, 4, 6, 1, 3, 5, 7]].unflatten(-1, (4, 2))          # nibbles in order, two to a byte
    return (code[..., 0] | code[..., 1] << 4).flatten(-3), torch.cat([scale, bias], -1).flatten(-2)


def _pages(count, layers, case, g):
    """Pages of rows as a layer makes them: normed keys with a few strong dims, normed values."""
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    strength = torch.exp(0.4 * torch.randn(dim, generator=g, device="cuda"))
    bits = case.get("bits", 16)
    if bits == 16:
        pages = torch.empty(layers, count, kv, 2, page, dim, dtype=torch.bfloat16, device="cuda")
    else:
        pages = torch.empty(layers, count, kv, 2, page * _row_bytes(case), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 28) // (kv * 2 * page * dim))
    for layer in range(layers):
        for a in range(0, count, step):
            n = min(step, count - a)
            x = torch.randn(n, kv, 2, page, dim, generator=g, device="cuda")
            x[:, :, 0] *= strength
            if bits == 16:
                pages[layer, a:a + n] = x
            else:
                codes, pairs = _quantised(x)
                pages[layer, a:a + n, ..., : page * dim // 2] = codes.flatten(-2)
                pages[layer, a:a + n, ..., page * dim // 2:] = pairs.contiguous().view(torch.uint8).flatten(-2)
    return pages, strength


def _package():
    import __graft_entry__

    return __graft_entry__.load_package()


def _handles(s, case):
    """The cache and the batch that a user's program keeps."""
    fm = _package()
    s["cache"] = fm.PagedKVCache.over(s["pages"], s["table"], s["lens"], s["refs"], kv_heads=case["kv_heads"], head_dim=case["dim"],
                                      page_size=case["page"], bits=case.get("bits", 16))
    if "q_start" in s:
        s["batch"] = fm.PagedBatch(s["seqs"], s["q_start"], s["kv_len"], tokens=s["tokens"], max_new=s["max_new"])
    if "theta" in case:
        s["norm"] = fm.QKNormRope(s["q_norm"], s["k_norm"], rope_dims=case["rope"], rope_theta=case["theta"])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = random.Random(seed)
    s = {"case": case}
    if case["op"] == "compact":
        live = _live(case)
        r.shuffle(live)
        table, refs = [live[i::case["seqs"]] for i in range(case["seqs"])], [0] * case["pages"]
        for p in live:
            refs[p] = 1
        width = max(len(t) for t in table) + 1
        s["lens"] = _ints([len(t) * case["page"] for t in table])
        s["table0"] = _ints([t + [-1] * (width - len(t)) for t in table])
        s["refs0"] = _ints(refs)
        s["table"], s["refs"] = s["table0"].clone(), s["refs0"].clone()
        s["pages"], _ = _pages(case["pages"], case["layers"], case, g)
    else:
        lens = _lengths(case)
        new = _new(case) if "new" in case else [1] * len(lens)
        held = [_seen(n, m, case) for n, m in zip(lens, new)]
        children = case.get("children", 0)
        count = sum(map(len, held)) + children + case.get("spare", 3)
        ids = list(range(count))
        r.shuffle(ids)
        rows = len(lens) + children + 2
        order = list(range(rows))  # rows of the table that the sequences have
        r.shuffle(order)
        width = max(_blocks(n, case) for n in lens) + 2
        table, refs, all_lens = [[-1] * width for _ in range(rows)], [0] * count, [0] * rows
        for i, blocks in enumerate(held):
            for b in blocks:
                table[order[i]][b] = ids.pop()
                refs[table[order[i]][b]] = 1
            all_lens[order[i]] = lens[i]
        s["table"], s["refs"], s["lens"] = _ints(table), _ints(refs), _ints(all_lens)
        layers = case.get("layers", 1)
        s["pages"], strength = _pages(count, layers, case, g)
        if case["op"] == "fork":
            s["from"] = _ints([order[i % len(lens)] for i in range(children)])
            s["to"] = _ints([order[len(lens) + i] for i in range(children)])
        else:
            s["tokens"], s["max_new"] = sum(new), max(new)
            s["seqs"], s["kv_len"] = _ints(order[: len(lens)]), _ints(lens)
            s["q_start"] = _ints([sum(new[:i]) for i in range(len(new) + 1)])
            h, kv, dim = case["heads"], case["kv_heads"], case["dim"]
            if case["op"] == "attend":
                s["q"] = (torch.randn(s["tokens"], h, dim, generator=g, device="cuda") * strength.reciprocal()).bfloat16()
                s["scale"] = 1.5 * dim ** -0.5
            else:
                s["q"], s["k"], s["v"] = (torch.randn(s["tokens"], n, dim, generator=g, device="cuda").bfloat16() for n in (h, kv, kv))
                s["q_norm"], s["k_norm"] = (torch.exp(0.3 * torch.randn(dim, generator=g, device="cuda")).bfloat16() for _ in range(2))
                if case["shared"]:
                    s["v"] = None
    if own:
        _handles(s, case)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------


def _rows_at(s, page, slot, ok):
    """K and V of positions [sequences, keys] as 32-bit values; zeros where there is no row."""
    case, dim = s["case"], s["case"]["dim"]
    if case["bits"] == 16:
        kv = s["pages"][0][page, :, :, slot].float()                           # [B, N, kv, 2, dim]
    else:
        size = case["page"] * dim // 2
        codes = s["pages"][0, ..., :size].unflatten(-1, (case["page"], dim // 2))[page, :, :, slot]
        pairs = s["pages"][0, ..., size:].unflatten(-1, (case["page"], dim // 16))[page, :, :, slot]
        pairs = pairs.contiguous().view(torch.bfloat16).float().unflatten(-1, (dim // 64, 2))
        nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (8, dim // 64, 8))
        code = nibbles[..., [0, 4, 1, 5, 2, 6, 3, 7]].transpose(-3, -2).flatten(-2).float()  # [..., group, 64]
        kv = (code * pairs[..., 0:1] + pairs[..., 1:2]).flatten(-2)
    kv = torch.where(ok[:, :, None, None, None], kv, 0.0)
    return kv[:, :, :, 0].transpose(1, 2), kv[:, :, :, 1].transpose(1, 2)      # [B, kv, N, dim]


def _plain_attend(s):
    case, page = s["case"], s["case"]["page"]
    window, sinks, kv_heads = case["window"], case["sinks"], case["kv_heads"]
    share = case["heads"] // kv_heads
    start, size = s["q_start"][:-1].long(), s["kv_len"].long()
    first = size - (s["q_start"][1:] - s["q_start"][:-1])                       # position of each sequence's first query
    at = torch.arange(_span(case), device="cuda")
    low = (first - window + 1).clamp(min=sinks) if window else torch.zeros_like(first)
    pos = torch.where(at < sinks, at, low[:, None] + at - sinks) if window else at.expand(len(first), -1)
    entry = torch.gather(s["table"][s["seqs"].long()], 1, (pos // page).clamp(max=s["table"].shape[1] - 1)).long()
    ok = (pos < size[:, None]) & (entry >= 0)
    k, v = _rows_at(s, entry.clamp(min=0), pos % page, ok)
    i = torch.arange(s["max_new"], device="cuda")
    q = s["q"].float()[(start[:, None] + i).clamp(max=s["tokens"] - 1)]         # [B, new, heads, dim]
    q = q.unflatten(2, (kv_heads, share)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [B, kv, share * new, dim]
    p = first[:, None] + i
    see = ok[:, None] & (pos[:, None] <= p[..., None])
    if window:
        see &= (pos[:, None] > p[..., None] - window) | (pos[:, None] < sinks)
    score = (q @ k.transpose(-1, -2) * s["scale"]).unflatten(2, (share, -1))
    score = score.masked_fill(~see[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    e = torch.exp(score - torch.where(top == float("-inf"), 0.0, top))
    total = e.sum(-1, keepdim=True)
    out = (e.flatten(2, 3) @ v).unflatten(2, (share, -1)) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).flatten(2, 3)                              # [B, new, heads, dim]
    token = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["q_start"].long(), token, right=True) - 1
    return out[b, token - start[b]].bfloat16()


def _plain_norm(x, weight=None):
    x = x.float()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    return x if weight is None else x * weight.float()


def _plain_turn(x, pos, case):
    half = case["rope"] // 2
    rate = torch.exp2(-torch.arange(half, device="cuda", dtype=torch.float64) / half * torch.log2(torch.tensor(case["theta"], dtype=torch.float64)).item())
    turn = pos[:, None, None] * rate  # whole positions times rates: 64 bits, since 32 lose the angle of a far token
    cos, sin = torch.cos(turn).float(), torch.sin(turn).float()
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)


def _plain_append(s):
    case = s["case"]
    token = torch.arange(s["tokens"], device="cuda")
    b = torch.searchsorted(s["q_start"].long(), token, right=True) - 1
    pos = s["kv_len"][b].long() - s["q_start"][b + 1] + token
    page = s["table"][s["seqs"][b].long(), pos // case["page"]].long()
    q = _plain_turn(_plain_norm(s["q"], s["q_norm"]), pos, case).bfloat16()
    k = _plain_turn(_plain_norm(s["k"], s["k_norm"]), pos, case).bfloat16()
    v = _plain_norm(s["k"] if s["v"] is None else s["v"]).bfloat16()
    s["pages"][0][page, :, :, pos % case["page"]] = torch.stack([k, v], 2)
    return {"q": q, "pages": s["pages"]}


def _plain_fork(s):
    case, page = s["case"], s["case"]["page"]
    src, dst = s["from"].long(), s["to"].long()
    one = torch.ones((), dtype=torch.int32, device="cuda")
    old = s["table"][dst]
    s["refs"].index_put_((old[old >= 0].long(),), -one, accumulate=True)
    rows, size = s["table"][src], s["lens"][src].long()
    part = size % page != 0
    free = torch.nonzero(s["refs"] == 0)[:, 0]
    fresh = free[part.long().cumsum(0) - 1]                                    # the lowest free pages, in the pairs' order
    last = size // page
    was = rows[torch.arange(len(src), device="cuda"), last].long()
    rows[torch.arange(len(src), device="cuda")[part], last[part]] = fresh[part].int()
    s["refs"].index_put_((rows[rows >= 0].long(),), one, accumulate=True)
    s["table"][dst], s["lens"][dst] = rows, s["lens"][src]
    s["pages"][:, fresh[part]] = s["pages"][:, was[part]]
    return {k: s[k] for k in ("pages", "table", "lens", "refs")}


def _plain_compact(s):
    live = s["refs"] > 0
    n = live.sum()
    ids = torch.arange(len(live), device="cuda")
    src, dst = torch.nonzero(live & (ids >= n))[:, 0], torch.nonzero(~live & (ids < n))[:, 0]
    to = ids.clone()
    to[src] = dst
    s["table"][:] = torch.where(s["table"] >= 0, to[s["table"].clamp(min=0).long()], -1)
    s["refs"][dst] = s["refs"][src]
    s["refs"][src] = 0
    s["pages"][:, dst] = s["pages"][:, src]
    return {**{k: s[k] for k in ("pages", "table", "refs")}, "live": n.int().reshape(1)}


def run(s):
    op = s["case"]["op"]
    if op == "compact":  # the pool as it was: a second pass has the same pages to move
        s["table"].copy_(s["table0"])
        s["refs"].copy_(s["refs0"])
    if not own:
        return {"attend": _plain_attend, "append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}[op](s)
    if op == "attend":
        return s["cache"].attend(0, s["q"], s["batch"], window=s["case"]["window"], sinks=s["case"]["sinks"], scale=s["scale"])
    if op == "append":
        return {"q": s["cache"].append_qkv(0, s["q"], s["k"], s["v"], s["batch"], s["norm"]), "pages": s["pages"]}
    if op == "fork":
        s["cache"].fork(s["from"], s["to"])
        return {k: s[k] for k in ("pages", "table", "lens", "refs")}
    n = s["cache"].compact()
    return {**{k: s[k] for k in ("pages", "table", "refs")}, "live": n}


# ---- the same in 64 bits, one sequence after another ---------------------------------------------------------------


def _exact_row(pages, case, page, slot):
    """Rows [keys, kv, 2, dim] of one sequence in 64 bits."""
    dim = case["dim"]
    if case["bits"] == 16:
        return pages[0, page, :, :, slot].double()
    block = pages[0, page]                                                      # [keys, kv, 2, bytes]
    at = torch.arange(len(page), device="cuda")
    words = block[..., : case["page"] * dim // 2].reshape(len(page), case["kv_heads"], 2, case["page"], dim // 2)[at, :, :, slot]
    pairs = block[..., case["page"] * dim // 2:].contiguous().view(torch.bfloat16)
    pairs = pairs.reshape(len(page), case["kv_heads"], 2, case["page"], dim // 64, 2)[at, :, :, slot].double()
    words = words.contiguous().view(torch.int32).long()
    d = torch.arange(dim, device="cuda")
    word = (d % 64 // 8) * (dim // 64) + d // 64
    nibble = (d % 8 // 2) + 4 * (d % 2)
    code = (words[..., word] >> (4 * nibble)) & 15
    return code.double() * pairs[..., d // 64, 0] + pairs[..., d // 64, 1]


def _exact_attend(s):
    case, out = s["case"], torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    share = case["heads"] // case["kv_heads"]
    starts, sizes, rows = s["q_start"].tolist(), s["kv_len"].tolist(), s["seqs"].tolist()
    for b, n in enumerate(sizes):
        for a in range(starts[b], starts[b + 1], 512):                          # a few queries at once
            z = min(starts[b + 1], a + 512)
            p = torch.arange(a, z, device="cuda") + (n - starts[b + 1])
            low = max(0, int(p[0]) - case["window"] + 1) if case["window"] else 0
            keys = sorted(set(range(min(case["sinks"], n)) if case["window"] else ()) | set(range(low, int(p[-1]) + 1)))
            j = torch.tensor(keys, device="cuda")
            page = s["table"][rows[b]].long()[j // case["page"]]
            kv = _exact_row(s["pages"], case, page.clamp(min=0), j % case["page"])
            see = (j <= p[:, None]) & (page >= 0)
            if case["window"]:
                see &= (p[:, None] - j < case["window"]) | (j < case["sinks"])
            k, v = (kv[:, :, i].repeat_interleave(share, 1) for i in (0, 1))
            w = torch.einsum("qhd,nhd->hqn", s["q"][a:z].double(), k) * s["scale"]
            w = torch.softmax(w.masked_fill(~see, float("-inf")), -1).nan_to_num(0.0)
            out[a:z] = torch.einsum("hqn,nhd->qhd", w, v)
    return out


def _exact_append(s):
    case, dim, half = s["case"], s["case"]["dim"], s["case"]["rope"] // 2
    pages = s["pages"].double()
    starts, sizes, rows = s["q_start"].tolist(), s["kv_len"].tolist(), s["seqs"].tolist()
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")

    def normed(x, w):
        x = x.double()
        x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / dim + 1e-6)
        return x if w is None else x * w.double()

    def turned(x, p):
        angle = p[:, None].double() * case["theta"] ** (-torch.arange(half, device="cuda").double() / half)
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle)[:, None]
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    for b, n in enumerate(sizes):
        a, z = starts[b], starts[b + 1]
        p = torch.arange(n - (z - a), n, device="cuda")
        q[a:z] = turned(normed(s["q"][a:z], s["q_norm"]), p)
        page = s["table"][rows[b]].long()[p // case["page"]]
        pages[0, page, :, 0, p % case["page"]] = turned(normed(s["k"][a:z], s["k_norm"]), p)
        pages[0, page, :, 1, p % case["page"]] = normed((s["k"] if s["v"] is None else s["v"])[a:z], None)
    return {"q": q, "pages": pages}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attend":
        return _exact_attend(s)
    if case["op"] == "append":
        return _exact_append(s)
    if case["op"] == "fork":  # moved bits and whole numbers: pages as they are, by walking the pairs one by one
        table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
        pairs, moves = list(zip(s["from"].tolist(), s["to"].tolist())), []
        for _, d in pairs:
            for p in table[d]:
                refs[p] -= p >= 0
            table[d], lens[d] = [-1] * len(table[d]), 0
        for a, d in pairs:
            table[d], lens[d] = list(table[a]), lens[a]
            if lens[a] % case["page"]:
                b = lens[a] // case["page"]
                table[d][b] = -1
        free = iter([p for p, n in enumerate(refs) if n == 0])
        for a, d in pairs:
            if lens[a] % case["page"]:
                b = lens[a] // case["page"]
                table[d][b] = next(free)
                moves.append((table[a][b], table[d][b]))
            for p in table[d]:
                refs[p] += p >= 0
        for a, d in moves:
            s["pages"][:, d] = s["pages"][:, a]
        return {"pages": s["pages"].double() if s["pages"].numel() < 2e9 else None, "table": _ints(table), "lens": _ints(lens), "refs": _ints(refs)}
    refs = s["refs"].tolist()
    live = [p for p, n in enumerate(refs) if n]
    holes, to = [p for p in range(len(live)) if not refs[p]], {}
    for p, d in zip([p for p in live if p >= len(live)], holes):
        s["pages"][:, d] = s["pages"][:, p]
        to[p], refs[d], refs[p] = d, refs[p], 0
    table = [[to.get(p, p) for p in row] for row in s["table"].tolist()]
    return {"pages": s["pages"].double() if s["pages"].numel() < 2e9 else None, "table": _ints(table), "refs": _ints(refs), "live": _ints([len(live)])}

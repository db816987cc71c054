"""Many sequences over paged KV caches: prompts of different lengths in one step,
decodes, a fork, pages given back, compaction.

    python examples/paged_serving.py [--bits 16|4] [--steps 24]

The decoder is a small one of random weights with the two kinds of layer that the
framework's models mix: sliding layers (more kv heads, smaller heads, a window
whose first positions stay visible) and full layers (values are the raw keys, part
of a head is rotated).  Each kind has a cache of its own, since a cache's pages
have one shape.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
from __graft_entry__ import load_package  # noqa: E402

fm = load_package()

HIDDEN, HEADS, VOCAB = 512, 8, 2048
KINDS = {  # kv heads, head dim, window, sinks, rotated dims, theta
    "sliding": (4, 256, 64, 4, 256, 1e4),
    "full": (1, 512, None, 0, 128, 1e6),
}


class Layer:
    def __init__(self, kind: str, device, gen):
        self.kind = kind
        kv_heads, dim, self.window, self.sinks, rope, theta = KINDS[kind]

        def linear(n_out, n_in):
            w = torch.randn(n_out, n_in, generator=gen, device=device) * n_in ** -0.5
            return fm.QuantizedLinear.from_float(w, bits=8)

        self.q, self.k = linear(HEADS * dim, HIDDEN), linear(kv_heads * dim, HIDDEN)
        self.v = linear(kv_heads * dim, HIDDEN) if kind == "sliding" else None
        self.o = linear(HIDDEN, HEADS * dim)
        ones = torch.ones(dim, device=device)
        self.norm = fm.QKNormRope(ones, ones, rope, theta)
        self.kv_heads, self.dim = kv_heads, dim


class Server:
    """Sequences are table rows 0 .. max_seqs - 1, in both caches alike."""

    def __init__(self, kinds=("sliding", "full", "sliding", "full"), bits=16, pages=256, max_seqs=8, max_blocks=64,
                 page_size=16, device="cuda", seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)
        self.layers = [Layer(k, device, gen) for k in kinds]
        self.embedding, self.head = (
            fm.QuantizedLinear.from_float(torch.randn(VOCAB, HIDDEN, generator=gen, device=device), bits=8) for _ in range(2))
        self.caches = {}
        for kind, (kv_heads, dim, *_) in KINDS.items():
            n = sum(x.kind == kind for x in self.layers)
            if n:
                self.caches[kind] = fm.PagedKVCache(n, kv_heads, dim, pages, max_seqs, max_blocks, page_size, bits, device)

    def step(self, seqs, ids):
        """ids[i]: the new tokens of sequence seqs[i].  The logits after each
        sequence's last one."""
        new = [len(x) for x in ids]
        batch = {kind: cache.reserve(seqs, new) for kind, cache in self.caches.items()}
        flat = torch.tensor([t for x in ids for t in x], dtype=torch.int32, device=self.embedding.weight.device)
        x = self.embedding.embed(flat).float()
        at = dict.fromkeys(self.caches, 0)  # the layer's number in its cache
        for layer in self.layers:
            cache, b, i = self.caches[layer.kind], batch[layer.kind], at[layer.kind]
            at[layer.kind] += 1
            h = torch.nn.functional.rms_norm(x, (HIDDEN,)).bfloat16()
            q = layer.q(h).view(-1, HEADS, layer.dim)
            k = layer.k(h).view(-1, layer.kv_heads, layer.dim)
            v = layer.v(h).view(-1, layer.kv_heads, layer.dim) if layer.v is not None else None
            q = cache.append_qkv(i, q, k, v, b, layer.norm)
            y = cache.attend(i, q, b, layer.window, layer.sinks, layer.dim ** -0.5)
            x = x + layer.o(y.view(len(flat), -1)).float()
        last = torch.tensor(new, device=x.device).cumsum(0) - 1
        return self.head(torch.nn.functional.rms_norm(x[last], (HIDDEN,)).bfloat16())

    def decode(self, seqs, logits, steps):
        """Greedy; the tokens of every sequence and the logits that follow them."""
        out = [[] for _ in seqs]
        for _ in range(steps):
            ids = logits.argmax(-1).tolist()
            for o, t in zip(out, ids):
                o.append(t)
            logits = self.step(seqs, [[t] for t in ids])
        return out, logits

    def fork(self, parents, children):
        for cache in self.caches.values():
            cache.fork(parents, children)

    def release(self, free=(), trim=()):
        """Sequences that are done, and pages that the window has left behind."""
        for kind, cache in self.caches.items():
            if free:
                cache.free(free)
            window, sinks = KINDS[kind][2:4]
            if trim and window:
                cache.trim(trim, window, sinks)

    def compact(self):
        """Live pages to the front; how many there are, by kind."""
        return {kind: int(cache.compact()) for kind, cache in self.caches.items()}

    def check(self):
        for kind, cache in self.caches.items():
            if int(cache.refused):
                raise RuntimeError(f"{kind}: {int(cache.refused)} requests found no page")
            if cache.status() != fm.FMOE_OK:
                raise RuntimeError(f"{kind}: a wait on the device gave up")


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--bits", type=int, default=16, choices=(16, 4))
    p.add_argument("--steps", type=int, default=24)
    a = p.parse_args(argv)
    server = Server(bits=a.bits)
    gen = torch.Generator().manual_seed(1)
    prompts = [torch.randint(VOCAB, (n,), generator=gen).tolist() for n in (150, 7, 61)]

    logits = server.step([0, 1, 2], prompts)                  # three prompts, one step
    tokens, logits = server.decode([0, 1, 2], logits, a.steps)
    for i, t in enumerate(tokens):
        print(f"sequence {i}: {len(prompts[i])} prompt tokens, then {t}")

    server.fork([0, 0], [3, 4])                               # sequence 0 goes on in three ways
    best = logits[0].topk(3).indices.tolist()
    logits = server.step([0, 3, 4], [[t] for t in best])
    tokens, logits = server.decode([0, 3, 4], logits, a.steps)
    for seq, first, t in zip((0, 3, 4), best, tokens):
        print(f"sequence {seq}: {[first] + t}")

    server.release(free=[1, 4], trim=[0, 2, 3])
    print("pages in use:", server.compact())
    logits = server.step([0, 2, 3], [[1], [2], [3]])          # the moved pages, as before
    print("next tokens:", logits.argmax(-1).tolist())
    server.check()


if __name__ == "__main__":
    main()

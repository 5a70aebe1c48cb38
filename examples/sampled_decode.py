"""Sampling with drafted trees over a cache in 4 bits that holds a bounded number of rows.

tree_verify.py's small transformer of random weights, with a temperature: every step
stores the drafted nodes' keys and values in 4 bits (cache.store4), attends over them,
accepts the tokens that the model's probabilities and given random numbers accept
(cache.verify), moves the accepted rows together, and adds the attention weight that every row
got from the accepted nodes to what it has gathered (cache.row_weights). A sequence of
more than `budget` rows keeps the first, the latest, and of the others those of most weight
(cache.evict).

    python examples/sampled_decode.py
"""

import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
for path in (ROOT, ROOT / "examples"):
    if str(path) not in sys.path:
        sys.path.insert(0, str(path))

from spiral_amd import cache, ops  # noqa: E402
from tree_verify import DIM, HEADS, KV, LAYERS, PAGE, Model, Sequence, device, norm  # noqa: E402

SINKS, RECENT = 4, 32


class Model4(Model):
    """The model with its cache in 4 bits."""

    def __init__(self, pages, seed=0):
        super().__init__(pages, seed)
        self.k, self.v = (cache.empty4(pages, PAGE, KV, DIM, layers=LAYERS) for _ in range(2))

    def forward(self, tokens, positions, trees):
        """Logits [nodes, VOCAB], and each layer's queries and attention lse."""
        x, seen = self.embed[tokens] + self.place[positions], []
        where = trees["table"], trees["lens"], trees["cu"]
        for i in range(LAYERS):
            qkv = self.qkv[i](norm(x)).view(-1, HEADS + 2 * KV, DIM)
            q, k, v = qkv.split((HEADS, KV, KV), dim=1)
            cache.store4(k, v, self.k[i], self.v[i], *where)
            o, lse = cache.tree_attention(q, self.k[i], self.v[i], **trees)
            seen.append((q, lse))
            x = x + self.out[i](o.view(-1, HEADS * DIM))
            x = x + self.down[i](ops.glu(self.up[i](norm(x), torch.float32)))
        return self.head(norm(x), torch.float32), seen


def chain_masks(counts):
    """A word per node of chains of up to 64: itself and those in front of it."""
    bits = [(2 << i) - 1 for t in counts for i in range(t)]
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64, device="cuda")[:, None]


def step(model, seqs, lens, mass, gen, size, width, temperature, budget):
    """One pass: new tokens are appended to seqs; (lengths, masses) of the cache returned."""
    drafts, masks, positions = [], [], []
    for s, n in zip(seqs, lens):
        rows = s.placed  # tokens that have their rows, or had them
        if rows + 1 < len(s.tokens):  # a prompt, 64 tokens at a time: a chain
            tokens = s.tokens[rows:rows + 64]
            parents = list(range(-1, len(tokens) - 1))
        else:
            tokens, parents = s.draft(size, width)
        depth, bits = [], []
        for i, p in enumerate(parents):
            depth.append(0 if p < 0 else depth[p] + 1)
            bits.append((0 if p < 0 else bits[p]) | 1 << i)
        s.pages = model.pool.extend(s.pages, n + len(tokens))
        drafts.append((tokens, parents))
        masks += [b - (1 << 64) if b >> 63 else b for b in bits]
        positions += [rows + d for d in depth]
    counts = [len(t) for t, _ in drafts]
    first = [sum(counts[:i]) for i in range(len(counts) + 1)]
    columns = max(len(s.pages) for s in seqs)
    table = device([s.pages + [-1] * (columns - len(s.pages)) for s in seqs])
    trees = dict(table=table, lens=device(lens), cu=device(first), max_tree=max(counts),
                 mask=torch.tensor(masks, dtype=torch.int64, device="cuda")[:, None],
                 max_len=max(n + c for n, c in zip(lens, counts)))
    tokens = device([t for d, _ in drafts for t in d])
    logits, seen = model.forward(tokens, device(positions), trees)

    # A prompt's tokens are given: what verify says of them is not used.
    accept = torch.rand(len(tokens), generator=gen, device="cuda")
    sample = torch.rand(len(seqs), generator=gen, device="cuda")
    keep, kept, said = cache.verify(logits, tokens, trees["cu"], accept, sample, max_tree=max(counts),
                                    temperature=torch.full_like(sample, temperature),
                                    parents=device([p for _, d in drafts for p in d]))
    keep, kept, said = keep.cpu(), kept.tolist(), said.tolist()
    for i, (s, (given, _)) in enumerate(zip(seqs, drafts)):
        if s.placed + 1 < len(s.tokens):
            kept[i] = len(given)
            keep[i, :kept[i]] = torch.arange(kept[i], dtype=torch.int32)
            if s.placed + kept[i] == len(s.tokens):  # its last token: the next one is drawn
                last = (logits[first[i] + kept[i] - 1] / temperature).softmax(0)
                s.tokens.append(int(torch.multinomial(last, 1, generator=gen)))
        else:
            s.tokens += said[i][:kept[i]]
        s.placed += kept[i]
    path = torch.cat([first[i] + keep[i, :c] for i, c in enumerate(kept)]).cuda()
    cache.compact(model.k, model.v, table, trees["lens"], keep.cuda(), device(kept), DIM)

    # The accepted nodes are chains on their rows now.
    start = [sum(kept[:i]) for i in range(len(kept) + 1)]
    wide = trees["max_len"] - mass.size(1)
    if wide > 0:
        mass = torch.nn.functional.pad(mass, (0, wide))
    for i, (q, lse) in enumerate(seen):
        cache.row_weights(q[path], model.k[i], table, trees["lens"], device(start), chain_masks(kept), lse[path], mass,
                          max_len=trees["max_len"], max_tree=max(kept))
    lens = [n + c for n, c in zip(lens, kept)]
    if max(lens) > budget:
        keep, left, mass = cache.evict(mass, device(lens), budget, sinks=SINKS, recent=RECENT)
        cache.compact(model.k, model.v, table, torch.zeros_like(left), keep, left, DIM)
        lens = left.tolist()
        for s, n in zip(seqs, lens):
            whole = -(-n // PAGE)
            model.pool.release(s.pages[whole:])
            s.pages = s.pages[:whole]
    return lens, mass


def generate(count, size, width, temperature=0.7, budget=96, prompts=((7, 8, 9) * 12, range(20, 60)), pages=64, seed=1):
    """At least `count` tokens behind each prompt: (token lists, passes, rows held)."""
    model, gen = Model4(pages), torch.Generator(device="cuda").manual_seed(seed)
    seqs = [Sequence(p) for p in prompts]
    for s in seqs:
        s.placed = 0
    goal, lens, passes = [len(s.tokens) + count for s in seqs], [0] * len(seqs), 0
    mass = torch.zeros((len(seqs), 0), device="cuda")
    while any(len(s.tokens) < g for s, g in zip(seqs, goal)):
        lens, mass = step(model, seqs, lens, mass, gen, size, width, temperature, budget)
        passes += 1
    for s in seqs:
        model.pool.release(s.pages)
    assert model.pool.free_pages == pages
    return [s.tokens for s in seqs], passes, lens


def main():
    for size, width in ((1, 1), (16, 3)):
        generate(8, size, width)  # the first calls load the kernels
        torch.cuda.synchronize()
        t = time.perf_counter()
        tokens, passes, lens = generate(200, size, width)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
        print(f"trees of up to {size} nodes: 2 x 200 tokens in {passes} passes, {t * 1e3:.0f} ms, "
              f"{lens} rows held of {[len(x) - 1 for x in tokens]}")
    print("tokens:", *tokens[0][36:56], "...")


if __name__ == "__main__":
    main()

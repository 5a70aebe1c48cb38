"""Decoding with drafted trees: MXFP4 weights, a paged cache, forks.

A small transformer of random weights continues a prompt twice, from a fork. Every
step verifies a tree of drafted tokens in one pass: the tree's nodes go through the
4-bit projections together, write their keys and values behind the cached rows and
attend over them (cache.tree_attention); the longest drafted path that the model
agrees with is kept (cache.compact) and the rest of the rows is overwritten by the
next step. Drafts come from the pairs of tokens seen so far.

    python examples/tree_verify.py
"""

import sys
import time
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

from spiral_amd import TYPE_MXFP4, cache, ops  # noqa: E402

HIDDEN, HEADS, KV, DIM, FFN, VOCAB, LAYERS, PAGE = 512, 8, 2, 64, 1024, 512, 2, 16


class Linear:
    """A weight matrix in MXFP4; rows come in bf16 or, with both=True, are quantized too."""

    def __init__(self, n, k, gen, both=False):
        self.n, self.k, self.both = n, k, both
        w = torch.randn((n, k), generator=gen) * k ** -0.5
        self.w = ops.mxfp4_quantize(w.bfloat16().cuda())

    def __call__(self, x, dtype=torch.bfloat16):
        if self.both:
            return ops.mxfp4_mul_mat(self.w, self.n, self.k, ops.mxfp4_quantize(x), x.size(0), out_dtype=dtype)
        return ops.mul_mat(TYPE_MXFP4, self.w, self.n, self.k, x, out_dtype=dtype)


def norm(x):
    x = x.float()
    return (x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)).bfloat16()


class Model:
    def __init__(self, pages, seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.embed = torch.randn((VOCAB, HIDDEN), generator=gen).bfloat16().cuda()
        self.place = (0.3 * torch.randn((4096, HIDDEN), generator=gen)).bfloat16().cuda()
        self.qkv = [Linear((HEADS + 2 * KV) * DIM, HIDDEN, gen) for _ in range(LAYERS)]
        self.out = [Linear(HIDDEN, HEADS * DIM, gen) for _ in range(LAYERS)]
        self.up = [Linear(2 * FFN, HIDDEN, gen, both=True) for _ in range(LAYERS)]
        self.down = [Linear(HIDDEN, FFN, gen, both=True) for _ in range(LAYERS)]
        self.head = Linear(VOCAB, HIDDEN, gen)
        shape = (LAYERS, pages, PAGE, KV, DIM)
        self.k, self.v = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.pool = cache.PagePool(pages, PAGE)

    def forward(self, tokens, positions, rows, trees):
        """Logits [nodes, VOCAB]; rows (page ids, rows in them) is where the nodes'
        keys and values go, trees the arguments of tree_attention."""
        x = self.embed[tokens] + self.place[positions]
        for i in range(LAYERS):
            qkv = self.qkv[i](norm(x)).view(-1, HEADS + 2 * KV, DIM)
            self.k[i][rows], self.v[i][rows] = qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:]
            o, _ = cache.tree_attention(qkv[:, :HEADS], self.k[i], self.v[i], **trees)
            x = x + self.out[i](o.view(-1, HEADS * DIM))
            x = x + self.down[i](ops.glu(self.up[i](norm(x), torch.float32)))
        return self.head(norm(x), torch.float32)


class Sequence:
    """Tokens decoded so far; all but the last have their rows in the cache."""

    def __init__(self, tokens, pages=()):
        self.tokens, self.pages, self.seen = list(tokens), list(pages), {}

    def draft(self, size, width):
        """A tree of up to `size` nodes on the last token: (tokens, parents). Each node is
        followed by the tokens last seen behind its own, the newest first."""
        tokens, parents = [self.tokens[-1]], [-1]
        for a, b in zip(self.tokens, self.tokens[1:]):
            after = self.seen.setdefault(a, [])
            if b in after:
                after.remove(b)
            after.insert(0, b)
        at = 0
        while at < len(tokens) and len(tokens) < size:
            for t in self.seen.get(tokens[at], [])[:width]:
                if len(tokens) < size:
                    tokens.append(t)
                    parents.append(at)
            at += 1
        return tokens, parents


def device(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def step(model, seqs, cached, size, width):
    """One pass over a drafted tree of every sequence (the prompt's rows as a chain
    where they are not cached yet); new tokens are appended, `cached` lengths returned."""
    drafts, masks, page_ids, page_rows, positions = [], [], [], [], []
    for s, n in zip(seqs, cached):
        if n + 1 < len(s.tokens):  # a prompt: a chain
            tokens = s.tokens[n:]
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
        positions += [n + d for d in depth]
        page_ids += [s.pages[(n + i) // PAGE] for i in range(len(tokens))]
        page_rows += [(n + i) % PAGE for i in range(len(tokens))]
    counts = [len(t) for t, _ in drafts]
    columns = max(len(s.pages) for s in seqs)
    table = device([s.pages + [-1] * (columns - len(s.pages)) for s in seqs])
    lens = device(cached)
    trees = dict(table=table, lens=lens, cu=device([sum(counts[:i]) for i in range(len(counts) + 1)]),
                 mask=torch.tensor(masks, dtype=torch.int64, device="cuda")[:, None],
                 max_len=max(n + c for n, c in zip(cached, counts)), max_tree=max(counts))
    logits = model.forward(device([t for d, _ in drafts for t in d]), device(positions),
                           (device(page_ids).long(), device(page_rows).long()), trees)
    best = logits.argmax(-1).tolist()
    keep, at = [], 0
    for s, (tokens, parents), n in zip(seqs, drafts, cached):
        node = len(tokens) - 1 if n + 1 < len(s.tokens) else 0  # a prompt is kept whole
        kept = list(range(node + 1))
        s.tokens.append(best[at + node])
        while True:
            child = [i for i in range(node + 1, len(tokens)) if parents[i] == node and tokens[i] == s.tokens[-1]]
            if not child:
                break
            node = child[0]
            kept.append(node)
            s.tokens.append(best[at + node])
        keep.append(kept)
        at += len(tokens)
    most = max(len(k) for k in keep)
    return cache.compact(model.k, model.v, table, lens, device([k + [-1] * (most - len(k)) for k in keep]),
                         device([len(k) for k in keep])).tolist()


def generate(count, size, width, prompt=range(7, 40), pages=256):
    """`count` tokens behind the prompt, and as many of a fork of it that begins with
    another token: (token lists, passes)."""
    model = Model(pages)
    first = Sequence(prompt)
    cached = step(model, [first], [0], size, width)
    ids, src, dst = model.pool.fork(first.pages, cached[0])
    if src:
        cache.copy_pages(model.k, model.v, device(src), device(dst))
    other = Sequence(first.tokens[:-1] + [(first.tokens[-1] + 1) % VOCAB], ids)
    seqs, cached, passes, goal = [first, other], cached * 2, 1, len(first.tokens) + count
    while min(len(s.tokens) for s in seqs) < goal:
        cached = step(model, seqs, cached, size, width)
        passes += 1
    for s in seqs:
        model.pool.release(s.pages)
    assert model.pool.free_pages == pages
    return [s.tokens[:goal] for s in seqs], passes


def shortfall(tokens, pages=256):
    """How far each token behind the first stays under the largest logit of its place, in
    standard deviations, all of them scored in one pass without a cached row."""
    model, n = Model(pages), len(tokens)
    ids = model.pool.alloc(-(-n // PAGE))
    words = -(-n // 64)
    mask = [[(1 << min(max(i + 1 - 64 * w, 0), 64)) - 1 for w in range(words)] for i in range(n)]
    trees = dict(table=device([ids]), lens=device([0]), cu=device([0, n]), max_len=n, max_tree=n,
                 mask=torch.tensor([[b - (1 << 64) if b >> 63 else b for b in row] for row in mask], device="cuda"))
    at = torch.arange(n, device="cuda")
    logits = model.forward(device(tokens), at, (device(ids).long()[at // PAGE], at % PAGE), trees)[:-1]
    taken = logits.gather(1, device(tokens[1:]).long()[:, None])[:, 0]
    return (logits.amax(-1) - taken) / logits.std(-1)


def main():
    for size, width in ((1, 1), (16, 2)):
        generate(8, size, width)  # the first calls load the kernels
        torch.cuda.synchronize()
        t = time.perf_counter()
        tokens, passes = generate(200, size, width)
        torch.cuda.synchronize()
        t = time.perf_counter() - t
        print(f"trees of up to {size} nodes: 2 x 200 tokens in {passes} passes, {t * 1e3:.0f} ms")
    print("tokens:", *tokens[0][33:53], "...")
    print(f"at most {float(shortfall(tokens[0])[33:].max()):.2f} standard deviations under the largest logit")


if __name__ == "__main__":
    main()

"""Store, attention, verification, compaction, weights and eviction one after the other, as
decoding over a bounded cache in 4 bits makes them, every step against the same on the host: a
list of rows a sequence, and the tests' definitions of each call."""

import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from spiral_amd import cache
from test_cache import U, check, pack, plain
from test_cache4 import decode, encode
from test_evict import chosen, walk as weights
from test_verify import expected

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

HEADS, KV, DIM, PAGE, VOCAB = 6, 2, 64, 16, 300


class Host:
    """One layer's cache as lists of rows, keys and values [kv, dim], in the values they hold."""

    def __init__(self, seqs):
        self.rows = [[] for _ in range(seqs)]
        self.mass = [np.zeros(0) for _ in range(seqs)]

    def cached(self):
        return [len(r) for r in self.rows]


def drafts(rng, counts):
    parents, seen = [], np.zeros((sum(counts), 64), dtype=bool)
    at = 0
    for t in counts:
        for i in range(t):
            p = int(rng.integers(0, i)) if i else -1
            if i:
                seen[at + i] = seen[at + p]
            seen[at + i, i] = True
            parents.append(p)
        at += t
    return parents, seen


@pytest.mark.gpu
@pytest.mark.parametrize("drawn", [False, True])
def test_steps(cuda, drawn):
    rng, gen = np.random.default_rng(5), torch.Generator().manual_seed(5)
    seqs, budget = 3, 12
    host = Host(seqs)
    pool = cache.PagePool(40, PAGE)
    k, v = (cache.empty4(40, PAGE, KV, DIM) for _ in range(2))
    ids, mass = [[] for _ in range(seqs)], torch.zeros((seqs, 128), device=cuda)
    bound = [np.zeros(0) for _ in range(seqs)]
    evicted = False

    def device(x):
        return torch.tensor(x, dtype=torch.int32, device=cuda)

    for turn in range(9):
        counts = [int(rng.integers(1, 20)) for _ in range(seqs)]
        if turn == 0:
            counts[1] = 25
        parents, seen = drafts(rng, counts)
        if drawn:
            parents = [i - 1 for t in counts for i in range(t)]
            seen = np.concatenate([np.tril(np.ones((t, 64), dtype=bool)) for t in counts])
        lens, nodes = host.cached(), sum(counts)
        cu = [0] + np.cumsum(counts).tolist()
        ids = [pool.extend(i, n + t) for i, n, t in zip(ids, lens, counts)]
        width = max(len(i) for i in ids)
        table = device([i + [-1] * (width - len(i)) for i in ids])
        qkv = torch.randn((nodes, HEADS + 2 * KV, DIM), generator=gen).bfloat16()
        d = qkv.to(cuda)
        q, new = d[:, :HEADS], (d[:, HEADS:HEADS + KV], d[:, HEADS + KV:])
        where = table, device(lens), device(cu)
        cache.store4(*new, k, v, *where)
        held = [decode(*encode(x.double().numpy())) for x in (qkv[:, HEADS:HEADS + KV], qkv[:, HEADS + KV:])]
        drafted = [[(held[0][i], held[1][i]) for i in range(cu[s], cu[s + 1])] for s in range(seqs)]

        # Attention, over the lists laid out in pages in order.
        mask = pack(seen)
        need = [-(-(n + t) // PAGE) for n, t in zip(lens, counts)]
        flat = np.full((2, sum(need), PAGE, KV, DIM), np.nan)
        order = np.full((seqs, max(need)), -1, dtype=np.int32)
        at = 0
        for s in range(seqs):
            order[s, :need[s]] = np.arange(at, at + need[s])
            for r, row in enumerate(host.rows[s] + drafted[s]):
                flat[:, at + r // PAGE, r % PAGE] = row
            at += need[s]
        c = dict(q=qkv[:, :HEADS], k=torch.from_numpy(flat[0]), v=torch.from_numpy(flat[1]), table=torch.from_numpy(order),
                 lens=torch.tensor(lens, dtype=torch.int32), cu=torch.tensor(cu, dtype=torch.int32), mask=mask)
        most = max(n + t for n, t in zip(lens, counts))
        out, lse = cache.tree_attention(q, k, v, *where, mask.to(cuda), max_len=most, max_tree=max(counts))
        check((out, lse), plain(c))

        # Verification.
        logits = 1.5 * torch.randn((nodes, VOCAB), generator=gen)
        draft = logits + 0.7 * torch.randn((nodes, VOCAB), generator=gen) if drawn else None
        behind = [cu[s] + max(parents[i], 0) for s in range(seqs) for i in range(cu[s], cu[s + 1])]
        tokens = torch.multinomial(torch.softmax((draft if drawn else 3 * logits)[behind], 1), 1, generator=gen)[:, 0].int()
        e = dict(logits=logits, tokens=tokens, cu=c["cu"], draft=draft, accept=0.6 * torch.rand(nodes, generator=gen),
                 parents=None if drawn else torch.tensor(parents, dtype=torch.int32), sample=torch.rand(seqs, generator=gen),
                 temperature=torch.tensor([1.0, 0.5, 0.0]))
        g = {n: x.to(cuda) if torch.is_tensor(x) else x for n, x in e.items()}
        keep, kept, said = cache.verify(g["logits"], g["tokens"], g["cu"], g["accept"], g["sample"], max_tree=max(counts),
                                        temperature=g["temperature"], parents=g["parents"], draft=g["draft"])
        path, number, words = expected(e, seqs, max(counts))
        assert keep.tolist() == path and kept.tolist() == number and said.tolist() == words

        # The accepted rows together, and the weight that they gave.
        assert cache.compact(k, v, *where[:2], keep, kept, DIM).tolist() == [n + m for n, m in zip(lens, number)]
        counted = torch.zeros(nodes)
        for s in range(seqs):
            counted[[cu[s] + i for i in path[s][:number[s]]]] = 1.0
        start = mass.clone()
        # Weights by the tree's places, as rows lay before they moved: the moved rows' are gathered.
        want, tol, _ = weights(c, lse.cpu(), counted)
        moved = [np.concatenate([np.arange(n), n + np.array(path[s][:number[s]], dtype=int)]) for s, n in enumerate(lens)]
        chain = torch.tensor(np.concatenate([[0], np.cumsum(number)]), dtype=torch.int32, device=cuda)
        nodes_kept = torch.tensor([cu[s] + i for s in range(seqs) for i in path[s][:number[s]]], device=cuda)
        chains = pack(np.concatenate([np.tril(np.ones((m, 64), dtype=bool)) for m in number])).to(cuda)
        cache.row_weights(q[nodes_kept], k, table, where[1], chain, chains, lse[nodes_kept], mass, max_len=most, max_tree=max(number))
        got = (mass.double() - start.double()).cpu().numpy()
        for s in range(seqs):
            host.rows[s] += [drafted[s][i] for i in path[s][:number[s]]]
            n = len(host.rows[s])
            slack = tol[s, moved[s]] + 2 * U * (np.abs(start[s, :n].cpu().numpy()) + np.abs(want[s, moved[s]]))
            assert (np.abs(got[s, :n] - want[s, moved[s]]) <= slack).all() and (got[s, n:] == 0).all()

        # Eviction.
        before = mass.cpu().numpy()
        lens = host.cached()
        keep, kept, mass = cache.evict(mass, device(lens), budget, sinks=2, recent=5)
        stay = [chosen(before[s], lens[s], budget, 2, 5) for s in range(seqs)]
        assert [x[x >= 0].tolist() for x in keep.cpu().numpy()] == [x.tolist() for x in stay]
        cache.compact(k, v, table, torch.zeros_like(kept), keep, kept, DIM)
        for s in range(seqs):
            evicted = evicted or len(stay[s]) < lens[s]
            host.rows[s] = [host.rows[s][i] for i in stay[s]]
            pages = -(-len(stay[s]) // PAGE)
            pool.release(ids[s][pages:])
            ids[s] = ids[s][:pages]
        n = host.cached()
        rows = device([0] + np.cumsum(n).tolist())
        for which, t in enumerate((k, v)):
            got = cache.load4(t, table, torch.zeros_like(kept), rows, torch.empty((sum(n), KV, DIM), dtype=torch.bfloat16, device=cuda))
            assert np.array_equal(got.double().cpu().numpy(), np.stack([r[which] for s in range(seqs) for r in host.rows[s]]))
    assert evicted


@pytest.mark.gpu
@pytest.mark.parametrize("size,width", [(1, 1), (16, 3)])
def test_example(cuda, size, width):
    """Runs, holds no more rows than it may, and gives the same tokens again."""
    import sampled_decode
    tokens, passes, lens = sampled_decode.generate(40, size, width, budget=64)
    assert [len(t) >= n + 40 for t, n in zip(tokens, (36, 40))] == [True, True] and max(lens) <= 64
    assert all(0 <= x < 512 for t in tokens for x in t) and (size > 1 or passes == 40)
    assert sampled_decode.generate(40, size, width, budget=64)[0] == tokens

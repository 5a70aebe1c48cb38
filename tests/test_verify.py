"""Verification of drafted tokens against the definition, walked a node at a time in
float64, and the definition against the distribution that it has to give.

Tokens have to be equal. A token of the two sides differs only where a border of a running
sum, or a chance, lies within its rounding of the random number: sums of up to 2^17
terms of 64 bits, their exponentials within 2^-49, move a border by less than 2^-48 of the
sum, so that one in 2^31 draws from 2^17 equally likely tokens may differ.
"""

import ctypes

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_BF16, cache
from test_cache_arguments import as_device, no_launch  # noqa: F401

FLOATS = [torch.float32, torch.float16, torch.bfloat16]


# ---- the definition --------------------------------------------------------------------


def probabilities(logits, temperature):
    """None where a row holds a NaN, +infinity, or nothing."""
    z = logits.double().numpy()
    if np.isnan(z).any() or np.isposinf(z).any() or np.isneginf(z).all():
        return None
    if not temperature > 0:
        w = np.zeros(len(z))
        w[np.argmax(z)] = 1.0
        return w
    w = np.exp((z - z.max()) / float(np.float32(temperature)))
    return w / w.sum()


def draw(w, u):
    upto = np.cumsum(w)
    past = np.nonzero(upto > u * upto[-1])[0]
    return int(past[0]) if len(past) else int(np.nonzero(w > 0)[0][-1])


def walk(c, s, max_tree):
    """(path, tokens) of sequence s."""
    first, last = int(c["cu"][s]), int(c["cu"][s + 1])
    count = min(last - first, max_tree)
    if count <= 0:
        return [], []
    vocab = c["logits"].shape[1]
    t = 1.0 if c["temperature"] is None else float(c["temperature"][s])
    u = float(c["sample"][s])
    node, path, said = 0, [0], []
    parent = [i - 1 if c["parents"] is None else int(c["parents"][first + i]) for i in range(count)]
    while True:
        p = probabilities(c["logits"][first + node], t)
        children = [i for i in range(node + 1, count) if parent[i] == node]
        if p is None:
            return path, said + [-1]
        left, turned, after, w = 1.0, set(), None, p
        for i in children:
            x, a = int(c["tokens"][first + i]), float(c["accept"][first + i])
            known = 0 <= x < vocab
            if c["draft"] is not None:
                q = probabilities(c["draft"][first + node], t)
                if q is not None and known and a * q[x] < p[x]:
                    after = i
                elif q is not None:
                    w = np.maximum(p - q, 0.0)
                break
            chance = p[x] if known and x not in turned else 0.0
            if a * left < chance:
                after = i
                break
            left -= chance
            turned.add(x)
        if after is None:
            if turned:
                w = p.copy()
                w[[x for x in turned if 0 <= x < vocab]] = 0.0
            return path, said + [draw(w if w.sum() > 0 else p, u)]
        node = after
        path.append(node)
        said.append(int(c["tokens"][first + node]))


def expected(c, seqs, max_tree):
    keep, kept, tokens = [], [], []
    for s in range(seqs):
        path, said = walk(c, s, max_tree)
        keep.append(path + [-1] * (max_tree - len(path)))
        tokens.append(said + [-1] * (max_tree - len(said)))
        kept.append(len(path))
    return keep, kept, tokens


def make(counts, vocab, dtype, draft, seed=0, temps=(0.7, 0.0, 1.0, 2.0, 0.05), chain=False, spread=2.0):
    gen, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    nodes, seqs = sum(counts), len(counts)
    logits = (spread * torch.randn((nodes, vocab), generator=gen)).to(dtype)
    q = (logits.float() + torch.randn((nodes, vocab), generator=gen)).to(dtype) if draft else None
    parents, tokens, at = [], [], 0
    for s, t in enumerate(counts):
        for i in range(t):
            p = i - 1 if draft or chain or rng.random() < 0.3 else int(rng.integers(0, i)) if i else -1
            parents.append(p)
            row = (q if draft else logits)[at + max(p, 0)].float()
            heat = max(temps[s % len(temps)], 0.05)
            g = -torch.log(-torch.log(torch.rand(vocab, generator=gen).clamp(min=1e-30)))
            tokens.append(int((row / heat + g).argmax()))
        at += t
    return dict(logits=logits, tokens=torch.tensor(tokens, dtype=torch.int32), accept=torch.rand(nodes, generator=gen),
                cu=torch.from_numpy(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)),
                parents=None if draft or chain else torch.tensor(parents, dtype=torch.int32), draft=q,
                sample=torch.rand(seqs, generator=gen),
                temperature=torch.tensor([temps[s % len(temps)] for s in range(seqs)], dtype=torch.float32))


def run(c, max_tree, dev, **kw):
    d = {n: t.to(dev) if torch.is_tensor(t) else t for n, t in c.items()}
    return cache.verify(d["logits"], d["tokens"], d["cu"], d["accept"], d["sample"], max_tree=max_tree,
                        temperature=d["temperature"], parents=d["parents"], draft=d["draft"], **kw)


def check(c, max_tree, dev, **kw):
    got = run(c, max_tree, dev, **kw)
    want = expected(c, c["sample"].numel(), max_tree)
    for g, w, name in zip(got, want, ("keep", "kept", "tokens")):
        assert g.tolist() == w, name
    return got


# ---- refusals (no device needed) --------------------------------------------------


def test_refusals(spiral_lib):
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4097)
    size = spiral_lib.spiral_draft_verify_workspace_bytes
    d = dict(type=TYPE_BF16, logits=p, ls=1000, draft=None, ds=0, nodes=6, vocab=1000, tokens=p, parents=p, cu=p, seqs=2,
             max_tree=4, accept=p, sample=p, temperature=p, keep=p, kept=p, out=p, ks=4, ws=p, wsb=1 << 20, stream=None)

    def call(**over):
        assert not set(over) - set(d)
        return spiral_lib.spiral_draft_verify(*{**d, **over}.values())

    assert call(type=8) == 6
    for bad in (dict(nodes=-1), dict(nodes=32768), dict(vocab=0), dict(vocab=1 << 25), dict(seqs=-1), dict(seqs=65536),
                dict(max_tree=1025), dict(max_tree=-1), dict(ls=999), dict(draft=p, parents=None, ds=999), dict(ks=3),
                dict(draft=p, ds=1000)):
        assert call(**bad) == 1, bad
    for bad in (dict(logits=None), dict(tokens=None), dict(cu=None), dict(accept=None), dict(sample=None), dict(keep=None),
                dict(kept=None), dict(out=None), dict(ws=None)):
        assert call(**bad) == 3, bad
    for bad in (dict(logits=odd), dict(tokens=odd), dict(cu=odd), dict(keep=odd), dict(ws=ctypes.c_void_p(4104)),
                dict(draft=odd, parents=None, ds=1000), dict(accept=odd), dict(temperature=odd)):
        assert call(**bad) == 2, bad
    assert call(wsb=size(6, 2, 1000, 0) - 1) == 7
    assert call(draft=p, parents=None, ds=1000, wsb=size(6, 2, 1000, 1) - 1) == 7
    assert call(seqs=0) == 0 and call(max_tree=0) == 0
    assert size(-1, 2, 1000, 0) == 0 and size(6, 2, 0, 0) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert call() == 4 and call(parents=None, temperature=None) == 4
        assert call(draft=p, parents=None, ds=1000) == 4 and call(nodes=0, logits=None, tokens=None, accept=None, ws=None, wsb=0) == 4


def test_wrapper_refusals(no_launch):  # noqa: F811
    c = make([2, 3], 11, torch.float32, False)
    ws = as_device(torch.empty(4096, dtype=torch.uint8))
    c = {n: as_device(t) if torch.is_tensor(t) else t for n, t in c.items()}

    def call(**over):
        d = {**c, **over}
        ids = as_device(torch.zeros(2, 4, dtype=torch.int32))
        kw = {"out": (ids, as_device(torch.zeros(2, dtype=torch.int32)), ids), **{n: over[n] for n in ("out", "workspace") if n in over}}
        return cache.verify(d["logits"], d["tokens"], d["cu"], d["accept"], d["sample"], max_tree=4,
                            temperature=d["temperature"], parents=d["parents"], draft=d["draft"], **{"workspace": ws, **kw})

    for bad, what in ((dict(logits=as_device(torch.zeros(5, 22)[:, ::2])), "contiguous"),
                      (dict(logits=as_device(torch.zeros(1, 11).expand(5, -1))), "overlap"),
                      (dict(logits=as_device(torch.zeros(5, 11, dtype=torch.float64))), "logits must be"),
                      (dict(logits=torch.zeros(5, 11)), "device"), (dict(draft=as_device(torch.zeros(5, 10))), "type and shape"),
                      (dict(draft=c["logits"]), "chains"), (dict(tokens=c["cu"]), "an entry for each node"),
                      (dict(accept=c["sample"]), "accept"), (dict(sample=as_device(torch.zeros(2, dtype=torch.float64))), "sample"),
                      (dict(temperature=torch.ones(2)), "temperature"), (dict(parents=as_device(c["parents"].long())), "parents"),
                      (dict(workspace=torch.empty(4096, dtype=torch.uint8)), "workspace"),
                      (dict(out=(as_device(torch.zeros(2, 3, dtype=torch.int32)),) * 3), "max_tree")):
        with pytest.raises(ValueError, match=what):
            call(**bad)


@pytest.mark.parametrize("draft", [False, True])
def test_sizes_that_are_not_taken(spiral_lib, draft):
    """Named where the workspace is asked for, which is of no use to them."""
    def size(nodes, vocab, seqs=2):
        logits = torch.empty((1, vocab), dtype=torch.bfloat16).expand(nodes, -1)
        return cache.verify_workspace(logits, seqs, 4, logits if draft else None).numel()

    for bad in ((32768, 9), (3, 0), (2, (1 << 24) + 1), (3, 9, 65536)):
        with pytest.raises(ValueError, match="32767 nodes"):
            size(*bad)
    assert size(32767, 9) >= 32767 * 16 and size(1, 1 << 24) >= 4096 * 16 and size(0, 9) >= 16


@pytest.mark.parametrize("draft", [False, True])
def test_definition_gives_the_targets_distribution(draft):
    """The first token's probabilities, from the walk's rule on a fine grid of its random
    numbers, are p. A grid of n midpoints in each of two numbers counts an area between
    curves that rise within 4 / n of it for each border."""
    gen = torch.Generator().manual_seed(1)
    vocab, n = 4, 400
    logits, q = torch.randn((3, vocab), generator=gen), torch.randn((3, vocab), generator=gen)
    p = probabilities(logits[0], 1.0)
    grid = (np.arange(n) + 0.5) / n
    got = np.zeros(vocab)
    if draft:
        chances = probabilities(q[0], 1.0)
        for x in range(vocab):
            taken = (grid * chances[x] < p[x]).mean()
            rest = np.maximum(p - chances, 0)
            got[x] += chances[x] * taken
            if taken < 1:
                for r in grid:
                    got[draw(rest, r)] += chances[x] * (1 - taken) / n
    else:
        for a in grid:  # children with tokens 2 and 0, the second's number independent
            if a < p[2]:
                got[2] += 1 / n
                continue
            second = (grid * (1 - p[2]) < p[0]).mean()
            got[0] += second / n
            rest = p.copy()
            rest[[2, 0]] = 0
            for x in range(vocab):
                got[x] += (1 - second) / n * rest[x] / rest.sum()
    assert np.abs(got - p).max() < 4 * 4 / n


# ---- on the device ------------------------------------------------------------------------


COUNTS = [[1], [2], [8], [3, 1, 5, 64, 2, 7], [130, 1], [1] * 70]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("vocab", [1, 7, 4096, 4097, 12289])
@pytest.mark.parametrize("draft", [False, True])
def test_walks(cuda, dtype, vocab, draft):
    for i, counts in enumerate(COUNTS):
        check(make(counts, vocab, dtype, draft, seed=vocab + i), max(counts), cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_large_vocabulary(cuda, draft):
    """Flat distributions, where every border counts."""
    for i in range(3):
        check(make([6, 9, 2, 5], 120007, torch.float32, draft, seed=i, spread=0.5, temps=(1.0, 3.0, 0.6, 1.5)), 9, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_chains_without_parents_and_temperature(cuda, draft):
    c = make([5, 1, 33], 501, torch.bfloat16, draft, seed=4, chain=True)
    check({**c, "temperature": None}, 33, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_trees_past_the_largest_and_empty(cuda, draft):
    """Nodes past max_tree are left out; sequences without a node keep none."""
    c = make([4, 0, 9, 0, 1], 333, torch.float32, draft, seed=6)
    c["cu"] = torch.tensor([0, 4, 4, 13, 13, 14], dtype=torch.int32)
    keep, kept, tokens = check(c, 6, cuda)
    assert kept[1] == 0 and kept[3] == 0 and (tokens[1] == -1).all()
    none = {n: t[:0] if torch.is_tensor(t) and n in ("logits", "tokens", "accept", "parents", "draft") else t for n, t in c.items()}
    none["cu"] = torch.zeros(6, dtype=torch.int32)
    keep, kept, tokens = run(none, 3, cuda)
    assert (keep == -1).all() and (tokens == -1).all() and (kept == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("accept,sample", [(0.0, 0.0), (1 - 2.0 ** -24, 1 - 2.0 ** -24), (0.0, 1 - 2.0 ** -24)])
def test_ends_of_the_random_numbers(cuda, draft, accept, sample):
    """0 takes whatever has a chance, the largest number only what is sure."""
    c = make([6, 20, 2, 3], 5001, torch.float32, draft, seed=8)
    c["logits"][:, 4000:] = -float("inf")  # tokens without a chance at the end
    if draft:
        c["draft"][:, 4000:] = -float("inf")
        c["tokens"].clamp_(max=3999)
    c["accept"].fill_(accept)
    c["sample"].fill_(sample)
    _, _, tokens = check(c, 20, cuda)
    assert int(tokens.max()) < 4000


@pytest.mark.gpu
def test_the_same_distribution_takes_every_token(cuda):
    c = make([9, 17], 2000, torch.bfloat16, True, seed=3, temps=(1.0, 0.5))
    c["draft"] = c["logits"].clone()
    c["accept"].fill_(1 - 2.0 ** -24)
    _, kept, _ = check(c, 17, cuda)
    assert kept.tolist() == [9, 17]


@pytest.mark.gpu
def test_nothing_left_of_the_difference(cuda):
    """A token outside the vocabulary behind equal distributions: drawn from p, in many chunks."""
    c = make([3] * 40, 20000, torch.float32, True, seed=7, temps=(1.0, 0.5))
    c["draft"] = c["logits"].clone()
    c["tokens"][torch.arange(1, 120, 3)] = 20000
    _, kept, _ = check(c, 3, cuda)
    assert (kept == 1).all()


@pytest.mark.gpu
def test_empty_trees_alone(cuda):
    c = make([1, 1], 9, torch.float32, False, seed=1)
    c["cu"].zero_()
    keep, kept, tokens = run(c, 0, cuda)
    assert keep.shape == tokens.shape == (2, 0) and kept.tolist() == [0, 0]


@pytest.mark.gpu
def test_tokens_that_are_none(cuda):
    """Outside the vocabulary, twice among siblings, all of them turned down."""
    c = make([9], 5, torch.float32, False, seed=5, temps=(1.0,))
    c["parents"] = torch.tensor([-1, 0, 0, 0, 0, 0, 0, 0, 0], dtype=torch.int32)
    for tokens, u in (([0, -1, 5, 7, 2, 2, 2 ** 30, 0, 0], 0.999), ([0, 0, 1, 2, 3, 4, 0, 1, 2], 0.99999), ([0, 3, 3, 3, 3, 3, 3, 3, 3], 0.9999)):
        c["tokens"], c["accept"] = torch.tensor(tokens, dtype=torch.int32), torch.full((9,), u)
        for r in (0.0, 0.3, 0.8, 0.99999):
            c["sample"] = torch.tensor([r])
            check(c, 9, cuda)


@pytest.mark.gpu
def test_largest_trees(cuda):
    """1024 nodes: a chain, and one node's children, nearly all of them turned down."""
    check(make([1024, 3], 60, torch.float32, False, seed=2, chain=True, spread=0.0), 1024, cuda)
    check(make([1024], 60, torch.bfloat16, True, seed=3, spread=0.1), 1024, cuda)
    c = make([1024], 2000, torch.float32, False, seed=5, temps=(1.0,))
    c["parents"] = torch.zeros(1024, dtype=torch.int32)
    c["tokens"] = torch.randperm(2000, generator=torch.Generator().manual_seed(1)).int()[:1024].contiguous()
    for u in (1 - 2.0 ** -24, 0.999, 0.9):
        c["accept"].fill_(u)
        check(c, 1024, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_largest_vocabulary(cuda, draft):
    check(make([2, 1], (1 << 24) - 5, torch.bfloat16, draft, seed=1, temps=(1.0, 0.8)), 2, cuda)


@pytest.mark.gpu
def test_parents_that_are_none(cuda):
    """Parents behind their nodes, past the tree or negative: such nodes are not reached."""
    c = make([7, 3], 50, torch.float32, False, seed=2, temps=(1.0, 0.0))
    c["parents"] = torch.tensor([5, 0, 2, 99, -7, 1, 0, -1, 1, 2 ** 30], dtype=torch.int32)
    c["accept"].fill_(0.0)
    check(c, 7, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), None])
def test_rows_without_a_distribution(cuda, draft, bad):
    """In the target's row the walk comes to, in one it does not, and in the draft's."""
    for node in range(4):
        for mine in ("logits", "draft") if draft else ("logits",):
            for greedy in (0.0, 1.0):
                c = make([4, 2], 9000, torch.float32, draft, seed=node, temps=(greedy, 1.0), chain=True)
                c["accept"].fill_(0.0)
                if draft and greedy:
                    c["draft"] = c["logits"].clone()
                if bad is None:
                    c[mine][node] = -float("inf")
                else:
                    c[mine][node, 8999 if node % 2 else 0] = bad
                _, _, tokens = check(c, 4, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
def test_strides_and_outputs(cuda, dtype):
    """Rows inside wider ones at odd addresses, given outputs of a wider layout, another stream."""
    c = make([5, 3], 4099, dtype, True, seed=9)
    d = dict(c)
    for n in ("logits", "draft"):
        wide = torch.full((8, 4099 + 6), float("nan"), dtype=dtype, device=cuda)
        wide[:, 3:4102] = c[n].to(cuda)
        d[n] = wide[:, 3:4102]
    ids = torch.full((2, 2, 11), 77, dtype=torch.int32, device=cuda)
    out = ids[0][:, :5], torch.empty(2, dtype=torch.int32, device=cuda), ids[1][:, :5]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(d, 5, cuda, out=out)
    side.synchronize()
    want = expected(c, 2, 5)
    assert got[0] is out[0] and [g.tolist() for g in got] == [*want]
    assert (ids[:, :, 5:] == 77).all()


@pytest.mark.gpu
def test_drawn_tokens_are_distributed_as_the_target(cuda):
    """One token drafted by another model, 20000 times: counts within five standard deviations."""
    gen = torch.Generator(device=cuda).manual_seed(11)
    n, vocab = 10000, 12
    p, q = torch.randn(vocab, generator=gen, device=cuda), torch.randn(vocab, generator=gen, device=cuda)
    chances = torch.softmax(p.double(), 0)
    for draft in (True, False):
        tokens = torch.zeros((n, 2), dtype=torch.int32, device=cuda)
        if draft:
            tokens[:, 1] = torch.multinomial(torch.softmax(q, 0), n, replacement=True, generator=gen).int()
        else:
            tokens[:, 1] = torch.randint(0, vocab, (n,), generator=gen, device=cuda).int()
        cu = 2 * torch.arange(n + 1, dtype=torch.int32, device=cuda)
        _, _, said = cache.verify(p.expand(2 * n, -1).contiguous(), tokens.view(-1), cu,
                                  torch.rand(2 * n, generator=gen, device=cuda), torch.rand(n, generator=gen, device=cuda), max_tree=2,
                                  draft=q.expand(2 * n, -1).contiguous() if draft else None)
        got = torch.bincount(said[:, 0].long(), minlength=vocab).double()
        assert ((got - n * chances).abs() <= 5 * (n * chances * (1 - chances)).sqrt()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("draft", [False, True])
def test_captured(cuda, draft):
    c = make([7, 3, 12], 9001, torch.bfloat16, draft, seed=1)
    d = {n: t.to(cuda) if torch.is_tensor(t) else t for n, t in c.items()}
    ws = cache.verify_workspace(d["logits"], 3, 12, d["draft"])

    def step():
        return cache.verify(d["logits"], d["tokens"], d["cu"], d["accept"], d["sample"], max_tree=12,
                            temperature=d["temperature"], parents=d["parents"], draft=d["draft"], workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        d["accept"].uniform_()
        d["sample"].uniform_()
        ws.fill_(0xFF)
        want = [t.clone() for t in step()]
        ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))

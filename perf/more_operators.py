"""Timed calls of a cache held in 4 bits, of drafts verified by random numbers, and of
eviction by accumulated attention weight.

The kinds of call, and what a program makes them for:

  store    new rows of keys and values quantized to MXFP4 into their pages, and read
           back as the values that the cache now holds
  attend   attention of a tree of drafted tokens over a paged cache held in 4 bits
  verify   which drafted tokens the target model's probabilities accept, for given
           random numbers, and the token drawn behind them: trees of given tokens, or
           chains drawn from a draft model's probabilities
  weigh    the attention weight that every cached row got from a step's queries, added to
           what it has gathered so far
  evict    the rows of every sequence that stay: the first, the latest, and of the others
           those of most weight

Where `own` is false a pass is written in elementary torch operations, where it
is true it is the framework's calls.

A page of a cache in 4 bits is, for each cached head, the codes of its rows (dim / 2
bytes a row, the even element of each pair in the low half of the byte), then the scale
bytes of each 32 elements, block after block: [page, dim / 2], [dim / 32, page].
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "fp4": 17 / 32}
# E2M1 values of the eight codes without a sign.
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # One token's keys and values on their way into the cache: the smallest call.
        dict(name="store_1x1", kind="store", seqs=1, rows=1, context=1000, kv=8, dim=128, page=16, dtype="bf16"),
        # Prompts of ragged lengths written into four layers' worth of heads.
        dict(name="store_8x2000", kind="store", seqs=8, rows=2000, context=300, kv=32, dim=128, page=64, dtype="f16"),
        # One sequence, one token: plain decoding over 4096 cached rows.
        dict(name="attend_1x1_4k", kind="attend", seqs=1, longest=4096, tree=1, heads=32, kv=8, dim=128, page=16,
             dtype="bf16"),
        # A serving batch of ragged lengths, drafts of up to 25 nodes.
        dict(name="attend_16x25_8k", kind="attend", seqs=16, longest=8192, tree=25, heads=32, kv=8, dim=128, page=32,
             dtype="f16"),
        # Decoding of a large batch, a token each: the cache's bytes decide.
        dict(name="attend_64x1_16k", kind="attend", seqs=64, longest=16384, tree=1, heads=32, kv=8, dim=128, page=64,
             dtype="bf16"),
        # Two long contexts, wide drafts, wide heads sharing one cached head.
        dict(name="attend_2x64_64k", kind="attend", seqs=2, longest=65536, tree=64, heads=8, kv=1, dim=256, page=64,
             dtype="bf16"),
        # One sequence's chain of seven tokens behind the last one, drawn from a draft model.
        dict(name="verify_1x8", kind="verify", seqs=1, tree=8, vocab=32000, dtype="bf16", draft=True),
        # A batch of trees of given tokens, an odd vocabulary.
        dict(name="verify_16x25", kind="verify", seqs=16, tree=25, vocab=100003, dtype="f32", draft=False),
        # The latest queries of one sequence weigh a short cache.
        dict(name="weigh_1x1_4k", kind="weigh", seqs=1, longest=4096, tree=1, heads=32, kv=8, dim=128, page=16,
             dtype="bf16", cache="bf16"),
        # A ragged batch, 32 queries each, over a cache in 4 bits.
        dict(name="weigh_16x32_8k", kind="weigh", seqs=16, longest=8192, tree=32, heads=32, kv=8, dim=128, page=32,
             dtype="f16", cache="fp4"),
        # Half of one short cache.
        dict(name="evict_1x4k", kind="evict", seqs=1, longest=4096, budget=2048, sinks=4, recent=256),
        # A quarter of many long ones.
        dict(name="evict_8x64k", kind="evict", seqs=8, longest=65536, budget=16384, sinks=16, recent=1024),
    ]


# ---- drawn cases ----------------------------------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["store", "attend", "attend", "verify", "verify", "weigh", "evict"])
    if kind == "evict":
        longest = _log(rng, 200, 131072)
        budget = max(1, int(longest * rng.uniform(0.1, 0.9)))
        sinks = min(rng.choice([0, 1, 4, 16]), budget)
        return dict(kind=kind, seqs=_log(rng, 1, 32), longest=longest, budget=budget, sinks=sinks,
                    recent=rng.randint(0, (budget - sinks) // 2))
    if kind == "verify":
        return dict(kind=kind, seqs=_log(rng, 1, 48), tree=_log(rng, 1, 48), vocab=_log(rng, 1000, 160000),
                    dtype=rng.choice(sorted(DTYPES)), draft=rng.random() < 0.5)
    kv, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([16, 32, 48, 64, 128, 256])
    dtype = rng.choice(["bf16", "f16"])
    if kind == "store":
        return dict(kind=kind, seqs=_log(rng, 1, 32), rows=_log(rng, 1, 2048), context=_log(rng, 1, 2000), kv=kv,
                    dim=dim, page=page, dtype=rng.choice(sorted(DTYPES)))
    case = dict(kind=kind, seqs=_log(rng, 1, 64), longest=_log(rng, 1, 65536), tree=_log(rng, 1, 64),
                heads=kv * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv=kv, dim=dim, page=page, dtype=dtype)
    if kind == "weigh":
        case["cache"] = rng.choice([dtype, "fp4"])
    return case


def _cost(case):
    w = work(case)
    return max(w["flops"] / 2.5e15, w["bytes"] / 8e12)


def _held(case):
    """Bytes that a case's inputs hold, in the larger of their forms."""
    if case["kind"] == "verify":
        return case["seqs"] * case["tree"] * case["vocab"] * (8 if case["draft"] else 4)
    if case["kind"] == "evict":
        return case["seqs"] * case["longest"] * 4
    rows = case["seqs"] * (case["longest"] + case["tree"] if "longest" in case else case["context"] + case["rows"])
    return 4 * (rows + case["seqs"] * case["page"]) * case["kv"] * case["dim"]


def draw(rng):
    limit = max(_cost(c) for c in listed())
    while True:
        case = _drawn(rng)
        if _cost(case) <= limit and _held(case) <= 5 << 30:
            return case


# ---- the 4-bit format -----------------------------------------------------------


def _encode(x):
    """Rows [..., dim] to codes [..., dim] (uint8 0 .. 15) and scale bytes [..., dim / 32]:
    the scale brings a block's largest value to [4, 8), codes are the nearest, ties to
    the even one, and end at 6."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(dim=-1, keepdim=True)
    _, e = torch.frexp(top)  # top = f 2^e, f in [0.5, 1)
    e = torch.where(top > 0, e - 3, -127).clamp(-127, 127)
    a = (b.abs() * torch.exp2(-e.double())).clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    q = torch.round(a / step) * step
    code = torch.where(q <= 2, 2 * q, torch.where(q <= 4, q + 2, 7.0)).to(torch.uint8)
    code = code + 8 * torch.signbit(b).to(torch.uint8)
    return code.flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _decode(code, scale, dtype=torch.float32):
    lut = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=dtype, device=code.device)
    s = torch.exp2(scale.to(dtype) - 127.0)
    return (lut[code.int()].unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _pages4(code, scale):
    """Codes [pages, page, kv, dim] and scales [pages, page, kv, blocks] as a cache in 4 bits."""
    pages, _, kv, _ = code.shape
    pair = code[..., 0::2] | code[..., 1::2] << 4
    pair, scale = pair.permute(0, 2, 1, 3), scale.permute(0, 2, 3, 1)
    return torch.cat([pair.reshape(pages, kv, -1), scale.reshape(pages, kv, -1)], dim=2).contiguous()


def _unpages4(cache, page, dim):
    """Codes and scales of pages of a cache in 4 bits."""
    pages, kv, _ = cache.shape
    pair = cache[..., :page * dim // 2].reshape(pages, kv, page, dim // 2)
    code = torch.stack([pair & 15, pair >> 4], dim=-1).flatten(-2).permute(0, 2, 1, 3)
    return code, cache[..., page * dim // 2:].reshape(pages, kv, dim // 32, page).permute(0, 3, 1, 2)


# ---- inputs ---------------------------------------------------------------------


def _gen(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rand(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _sizes(case):
    """Ragged lengths and new rows (or drafted nodes) of a batch, the first sequence's the longest."""
    rng = np.random.default_rng(case["seqs"] * 1000003 + case.get("dim", 7) * 1009 + case.get("page", 5))
    more = range(case["seqs"] - 1)
    if case["kind"] == "evict":
        return [case["longest"]] + [int(rng.integers(0, case["longest"] + 1)) for _ in more], None
    if case["kind"] == "store":
        return ([case["context"]] + [int(rng.integers(0, case["context"] + 1)) for _ in more],
                [case["rows"]] + [int(rng.integers(1, case["rows"] + 1)) for _ in more])
    counts = [case["tree"]] + [int(rng.integers(1, case["tree"] + 1)) for _ in more]
    if case["kind"] == "verify":
        return None, counts
    return [max(case["longest"] - case["tree"], 0)] + [int(rng.integers(0, case["longest"])) for _ in more], counts


def _table(need, gen):
    """A table of distinct page ids in random order: sequence s has need[s] of them."""
    total = int(sum(need)) + 3
    order = torch.randperm(total, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((len(need), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = order[at:at + c]
        at += c
    return table, total


def _parents(counts, rng, chain):
    """Parent of each node in its tree, -1 for the first."""
    out = []
    for t in counts:
        out += [-1] + [i - 1 if chain or rng.random() < 0.4 else int(rng.integers(0, i)) for i in range(1, t)]
    return out


def _cu(counts):
    return [0] + np.cumsum(counts).tolist()


def _cached(case, total, gen):
    """A layer's keys (or values), a few channels larger than the others as keys have them."""
    kv, dim, page = case["kv"], case["dim"], case["page"]
    channel = torch.exp(0.4 * _randn(gen, 1, 1, kv, dim))
    if case.get("cache", "fp4") != "fp4":
        return (_randn(gen, total, page, kv, dim) * channel).to(DTYPES[case["cache"]])
    step = max(1, (1 << 25) // (page * kv * dim))
    return torch.cat([_pages4(*_encode(_randn(gen, min(step, total - p), page, kv, dim) * channel))
                      for p in range(0, total, step)])


def _inputs(case, seed):
    gen, rng, kind = _gen(seed), np.random.default_rng(seed), case["kind"]
    lens, counts = _sizes(case)
    if kind == "evict":  # weight gathered: a long tail, the first rows far above it, some rows none
        mass = torch.exp(2.0 * _randn(gen, case["seqs"], case["longest"]) - 6.0)
        mass[:, :4] += 50.0
        return dict(mass=torch.where(_rand(gen, *mass.shape) < 0.02, torch.zeros_like(mass), mass), lens=_int32(lens),
                    host=lens)
    if kind == "verify":
        cu = _cu(counts)
        nodes, vocab, dt = cu[-1], case["vocab"], DTYPES[case["dtype"]]
        parents = _parents(counts, rng, case["draft"])
        first = torch.tensor([at for at, t in zip(cu, counts) for _ in range(t)], device="cuda")
        parent = _int32(parents)
        before = (first + parent.clamp(min=0)).long()
        logits = (2.5 * _randn(gen, nodes, vocab)).to(dt)
        temperature = torch.where(torch.arange(case["seqs"], device="cuda") % 4 == 3, 0.0,
                                  0.3 + 0.5 * _rand(gen, case["seqs"]))
        of = torch.tensor([s for s, t in enumerate(counts) for _ in range(t)], device="cuda")
        draft = (logits.float() + 0.5 * _randn(gen, nodes, vocab)).to(dt) if case["draft"] else None
        # Drawn from the draft model's probabilities behind the parent, or likely ones of the target's.
        noise = torch.empty((nodes, vocab), device="cuda").exponential_(generator=gen).log_().neg_()
        source = (draft if case["draft"] else logits)[before].float()
        tokens = (source + temperature[of, None].clamp(min=0.05) * noise).argmax(dim=1).int()
        return dict(logits=logits, tokens=tokens, cu=_int32(cu), parents=parent, draft=draft, accept=_rand(gen, nodes),
                    sample=_rand(gen, case["seqs"]), temperature=temperature, max_tree=max(counts), host=counts)
    cu, dt, kv, dim, page = _cu(counts), DTYPES[case["dtype"]], case["kv"], case["dim"], case["page"]
    table, total = _table([-(-(n + t) // page) for n, t in zip(lens, counts)], gen)
    s = dict(table=table, lens=_int32(lens), cu=_int32(cu), host=list(zip(lens, counts)),
             max_len=max(n + t for n, t in zip(lens, counts)), max_tree=max(counts))
    if kind == "store":
        column = torch.exp(0.5 * _randn(gen, 1, kv, dim))
        s.update(new=[(_randn(gen, cu[-1], kv, dim) * column).to(dt) for _ in range(2)],
                 cache=[torch.zeros((total, kv, page * dim * 17 // 32), dtype=torch.uint8, device="cuda") for _ in range(2)])
        return s
    anc, at = [], 0
    parents = _parents(counts, rng, False)
    for t in counts:
        for i in range(t):
            anc.append(1 << i | (anc[at + parents[at + i]] if i else 0))
        at += t
    s["mask"] = torch.tensor([a - (1 << 64) if a >> 63 else a for a in anc], dtype=torch.int64)[:, None].cuda()
    s["q"] = (1.5 * _randn(gen, cu[-1], case["heads"], dim)).to(dt)
    s["k"] = _cached(case, total, gen)
    if kind == "attend":
        s["v"] = _cached(case, total, gen)
    else:  # what attention left, and the weight gathered in earlier steps
        s["mass"] = torch.exp(_randn(gen, case["seqs"], s["max_len"]) - 4.0)
        s["lse"] = torch.cat([torch.cat([torch.logsumexp(z, dim=-1).permute(1, 2, 0).flatten(1) for z in [_scores(s, case, i, at)]])
                              for i, at in enumerate(cu[:-1])])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:  # the workspaces a program keeps
        from spiral_amd import cache
        if case["kind"] == "attend":
            s["ws"] = cache.tree_attention_workspace(s["q"], s["k"], case["seqs"], s["max_len"], s["max_tree"])
        if case["kind"] == "verify":
            s["ws"] = cache.verify_workspace(s["logits"], case["seqs"], s["max_tree"], s["draft"])
    return s


# ---- one pass -------------------------------------------------------------------


def _rows(cache, ids, case, n):
    """The first n rows of pages `ids` in 32 bits, [n, kv, dim]."""
    pages = cache[ids]
    if cache.dtype is torch.uint8:
        pages = _decode(*_unpages4(pages, case["page"], case["dim"]))
    return pages.flatten(0, 1)[:n].float()


def _scores(s, case, i, at):
    """Scores of sequence i's nodes from `at` on, -inf where a row is not seen: [kv, nodes, group, rows]."""
    n, t = s["host"][i]
    kv, dim, group = case["kv"], case["dim"], case["heads"] // case["kv"]
    k = _rows(s["k"], s["table"][i, :-(-(n + t) // case["page"])].long(), case, n + t).permute(1, 2, 0).contiguous()
    q = s["q"][at:at + t].float().view(t, kv, group, dim).permute(1, 0, 2, 3).reshape(kv, t * group, dim)
    z = torch.matmul(q, k).view(kv, t, group, n + t) * dim ** -0.5
    seen = (s["mask"][at:at + t, 0:1] >> torch.arange(t, device=q.device)) & 1
    z[..., n:].masked_fill_((seen == 0)[None, :, None, :], -math.inf)
    return z


def _store_plain(s):
    case, out = s["case"], []
    at = torch.cat([torch.arange(n, n + t, device="cuda") for n, t in s["host"]])
    seq = torch.cat([torch.full((t,), i, device="cuda") for i, (_, t) in enumerate(s["host"])])
    where = s["table"][seq, at // case["page"]].long()
    for new, cache in zip(s["new"], s["cache"]):
        code, scale = _encode(new)
        row, half = at % case["page"], case["page"] * case["dim"] // 2
        codes = cache[..., :half].unflatten(-1, (case["page"], -1))
        scales = cache[..., half:].unflatten(-1, (-1, case["page"]))
        codes[where, :, row] = code[..., 0::2] | code[..., 1::2] << 4
        scales[where, :, :, row] = scale
        pair = codes[where, :, row]
        out.append(_decode(torch.stack([pair & 15, pair >> 4], dim=-1).flatten(-2), scales[where, :, :, row],
                           torch.float64).to(new.dtype if new.dtype is not torch.float32 else torch.bfloat16))
    return out


def _attend_plain(s):
    case, q = s["case"], s["q"]
    heads, dim, kv = case["heads"], case["dim"], case["kv"]
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    at = 0
    for i, (n, t) in enumerate(s["host"]):
        z = _scores(s, case, i, at)
        v = _rows(s["v"], s["table"][i, :-(-(n + t) // case["page"])].long(), case, n + t).permute(1, 0, 2).contiguous()
        top = z.amax(dim=-1, keepdim=True)
        p = torch.exp(z - top)
        total = p.sum(dim=-1, keepdim=True)
        o = torch.matmul((p / total).view(kv, -1, n + t), v)
        out[at:at + t] = o.view(kv, t, heads // kv, dim).permute(1, 0, 2, 3).reshape(t, heads, dim).to(q.dtype)
        lse[at:at + t] = (top + torch.log(total))[..., 0].permute(1, 0, 2).reshape(t, heads)
        at += t
    return [out, lse]


def _weigh_plain(s):
    at = 0
    for i, (n, t) in enumerate(s["host"]):
        lse = s["lse"][at:at + t].view(t, s["case"]["kv"], -1).permute(1, 0, 2)
        s["mass"][i, :n + t] += torch.exp(_scores(s, s["case"], i, at) - lse[..., None]).sum(dim=(0, 1, 2))
        at += t
    return s["mass"]


def _probabilities(logits, temperature):
    """Softmax of rows / temperature in 64 bits: draws turn on single bits. 0 is the first of the largest."""
    z = logits.double()
    z = torch.exp((z - z.amax(dim=1, keepdim=True)) / torch.where(temperature > 0, temperature, 1.0).double()[:, None])
    z /= z.sum(dim=1, keepdim=True)
    best = torch.zeros_like(z).scatter_(1, logits.float().argmax(dim=1, keepdim=True), 1.0)
    return torch.where(temperature[:, None] > 0, z, best)


def _verify_plain(s):
    case = s["case"]
    seqs, width, vocab = case["seqs"], s["max_tree"], case["vocab"]
    first, count = s["cu"][:-1].long(), s["cu"].diff()
    every = torch.arange(seqs, device="cuda")
    of = torch.repeat_interleave(every, count)
    p = _probabilities(s["logits"], s["temperature"][of])
    q = _probabilities(s["draft"], s["temperature"][of]) if case["draft"] else None
    at = torch.zeros(seqs, dtype=torch.long, device="cuda")  # the node that the walk has come to
    stopped = torch.zeros(seqs, dtype=torch.bool, device="cuda")
    left = torch.ones(seqs, dtype=torch.float64, device="cuda")  # probability of what was not turned down there
    out = torch.zeros((seqs, vocab), dtype=torch.bool, device="cuda")
    keep = torch.full((seqs, width), -1, dtype=torch.int32, device="cuda")
    tokens, kept = keep.clone(), torch.ones(seqs, dtype=torch.long, device="cuda")
    keep[:, 0] = 0
    for i in range(1, width):
        node = (first + i).clamp(max=s["tokens"].numel() - 1)
        token = s["tokens"][node].long()
        tried = (i < count) & (s["parents"][node] == at) & ~stopped
        chance = p[first + at, token]
        if q is not None:
            taken = s["accept"][node].double() * q[first + at, token] < chance
        else:
            chance = torch.where(out[every, token], 0.0, chance)
            taken = s["accept"][node].double() * left < chance
        taken, failed = taken & tried, ~taken & tried
        if q is not None:
            stopped |= failed
        left = torch.where(taken, 1.0, torch.where(failed, left - chance, left))
        out[every, token] |= failed
        out &= ~taken[:, None]
        keep[every, kept.clamp(max=width - 1)] = torch.where(taken, i, keep[every, kept.clamp(max=width - 1)])
        tokens[every, kept - 1] = torch.where(taken, token.int(), tokens[every, kept - 1])
        at, kept = torch.where(taken, i, at), kept + taken
    rest = p[first + at]
    if q is not None:
        rest = torch.where(stopped[:, None], (rest - q[first + at]).clamp(min=0.0), rest)
    else:
        rest = torch.where(out, 0.0, rest)
    rest = torch.where(rest.sum(dim=1, keepdim=True) > 0, rest, p[first + at])
    upto = rest.cumsum(dim=1)
    drawn = torch.searchsorted(upto, s["sample"].double()[:, None] * upto[:, -1:], right=True)[:, 0]
    tokens[every, kept - 1] = drawn.clamp(max=vocab - 1).int()
    return [keep, kept.int(), tokens]


def _evict_plain(s):
    case, mass = s["case"], s["mass"]
    seqs, cols, budget = case["seqs"], case["longest"], case["budget"]
    pos, n = torch.arange(cols, device="cuda")[None, :], s["lens"][:, None]
    kept = torch.minimum(s["lens"], _int32(budget))
    value = torch.where((pos < case["sinks"]) | (pos >= n - case["recent"]), math.inf, mass)
    value = torch.where(pos < n, value, -math.inf)
    order = torch.sort(value, dim=1, descending=True, stable=True).indices
    stays = torch.zeros((seqs, cols), dtype=torch.bool, device="cuda").scatter_(1, order, pos < kept[:, None])
    rows = torch.sort(torch.where(stays, pos, cols), dim=1).values[:, :budget]
    on = rows < cols
    new = torch.zeros_like(mass)
    new[:, :rows.shape[1]] = torch.where(on, mass.gather(1, rows.clamp(max=cols - 1)), 0.0)
    return [torch.where(on, rows, -1).int(), kept, new]


def run(s):
    case = s["case"]
    kind = case["kind"]
    if not own:
        return dict(store=_store_plain, attend=_attend_plain, verify=_verify_plain, weigh=_weigh_plain,
                    evict=_evict_plain)[kind](s)
    from spiral_amd import cache
    if kind == "store":
        cache.store4(*s["new"], *s["cache"], s["table"], s["lens"], s["cu"])
        out = [torch.empty_like(x, dtype=x.dtype if x.dtype is not torch.float32 else torch.bfloat16) for x in s["new"]]
        for c, o in zip(s["cache"], out):
            cache.load4(c, s["table"], s["lens"], s["cu"], o)
        return out
    if kind == "attend":
        return list(cache.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["cu"], s["mask"],
                                         max_len=s["max_len"], max_tree=s["max_tree"], workspace=s["ws"]))
    if kind == "verify":
        return list(cache.verify(s["logits"], s["tokens"], s["cu"], s["accept"], s["sample"], max_tree=s["max_tree"],
                                 temperature=s["temperature"], parents=None if case["draft"] else s["parents"],
                                 draft=s["draft"], workspace=s["ws"]))
    if kind == "weigh":
        return cache.row_weights(s["q"], s["k"], s["table"], s["lens"], s["cu"], s["mask"], s["lse"], s["mass"],
                                 max_len=s["max_len"], max_tree=s["max_tree"])
    return list(cache.evict(s["mass"], s["lens"], case["budget"], sinks=case["sinks"], recent=case["recent"]))


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    kind = case["kind"]
    lens, counts = _sizes(case)
    if kind == "evict":
        return {"bytes": 4 * sum(lens) + case["seqs"] * 4 * (case["budget"] + case["longest"] + 2), "flops": 0}
    if kind == "verify":
        rows = sum(counts) + (sum(counts) - case["seqs"] if case["draft"] else 0)
        return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + 8 * case["seqs"] * max(counts), "flops": 0}
    width = case["kv"] * case["dim"]
    if kind == "store":  # the stored rows are read back as values
        n = 2 * sum(counts) * width
        return {"bytes": n * (SIZE[case["dtype"]] + 2 * SIZE["fp4"] + 2), "flops": 0}
    pairs = sum((n + t) * t for n, t in zip(lens, counts))  # of a query and a row
    rows, query = sum(lens) + sum(counts), sum(counts) * case["heads"]
    row, one = width * SIZE[case.get("cache", "fp4")], case["dim"] * SIZE[case["dtype"]]
    if kind == "attend":
        return {"bytes": 2 * rows * row + query * (2 * one + 4), "flops": 4 * pairs * case["heads"] * case["dim"]}
    return {"bytes": rows * (row + 8) + query * (one + 4), "flops": 2 * pairs * case["heads"] * case["dim"]}


# ---- the same in float64 --------------------------------------------------------


def _exact_e2m1(x):
    """Nearest E2M1 multiple of each block's scale, ties to the even code, by
    comparing with the borders between neighbouring values."""
    b = x.double().reshape(-1, 32)
    top = b.abs().max(dim=1, keepdim=True).values
    scale = torch.full_like(top, 2.0 ** -127)
    for e in range(-126, 128):  # the largest power of two with top / scale >= 4
        scale = torch.where(top >= 2.0 ** (e + 2), torch.full_like(scale, 2.0 ** e), scale)
    a, code = b.abs() / scale, torch.zeros(b.shape, dtype=torch.long, device=x.device)
    for c in range(7):
        border = (E2M1[c] + E2M1[c + 1]) / 2
        code += ((a >= border) if c % 2 else (a > border)).long()  # a tie goes to the even of c and c + 1
    v = torch.tensor(E2M1, dtype=torch.float64, device=x.device)[code]
    return (torch.where(b < 0, -v, v) * scale).reshape(x.shape)


def _exact_head(cache, table, pos, h, case):
    """Rows `pos` of cached head h, [rows, dim]."""
    page, dim = case["page"], case["dim"]
    where, row = table[pos // page].long(), pos % page
    if cache.dtype is not torch.uint8:
        return cache[where, row, h].double()
    flat, out = cache[:, h], torch.empty((pos.numel(), dim), dtype=torch.float64, device=cache.device)
    lut = torch.tensor(E2M1, dtype=torch.float64, device=cache.device)
    for d in range(dim):
        code = flat[where, row * (dim // 2) + d // 2].long() // (16 if d % 2 else 1) % 16
        scale = flat[where, page * dim // 2 + d // 32 * page + row].double() - 127
        out[:, d] = lut[code % 8] * torch.where(code >= 8, -1.0, 1.0) * torch.pow(2.0, scale)
    return out


def _exact_attention(s, case):
    """For each sequence: (sequence, nodes, cached head, its query heads, scores in 64 bits)."""
    mask, at, heads, kv = s["mask"][:, 0].tolist(), 0, case["heads"], case["kv"]
    for i, (n, t) in enumerate(s["host"]):
        pos = torch.arange(n + t, device="cuda")
        allowed = torch.tensor([[True] * n + [bool(mask[at + r] >> j & 1) for j in range(t)] for r in range(t)]).cuda()
        for h in range(kv):
            k = _exact_head(s["k"], s["table"][i], pos, h, case)
            for g in range(h * heads // kv, (h + 1) * heads // kv):
                z = s["q"][at:at + t, g].double() @ k.t() / math.sqrt(case["dim"])
                yield i, at, pos, h, g, torch.where(allowed, z, -math.inf)
        at += t


def _exact_verify(s, case):
    """A sequence at a time, children of a node one after the other."""
    width, vocab, at = s["max_tree"], case["vocab"], 0
    keep, kept, tokens = [], [], []
    for i, t in enumerate(s["host"]):
        temperature = float(s["temperature"][i])

        def weights(logits):
            z = logits.double()
            if temperature == 0:
                w = torch.zeros_like(z)
                w[int(torch.nonzero(z == z.max())[0])] = 1.0
                return w
            return torch.softmax(z / temperature, dim=0)

        node, path, said = 0, [0], []
        while True:
            p, after = weights(s["logits"][at + node]), None
            q = weights(s["draft"][at + node]) if case["draft"] else None
            for c in [c for c in range(node + 1, t) if int(s["parents"][at + c]) == node]:
                x, u = int(s["tokens"][at + c]), float(s["accept"][at + c])
                if u * (float(q[x]) if q is not None else float(p.sum())) < float(p[x]):
                    after = c
                    break
                before = p
                if q is not None:
                    p = torch.clamp(p - q, min=0)
                else:
                    p = p.clone()
                    p[x] = 0
                p = p if float(p.sum()) > 0 else before
            if after is None:
                break
            node = after
            path.append(node)
            said.append(int(s["tokens"][at + node]))
        upto = torch.cumsum(p, 0)
        said.append(min(int((upto <= float(s["sample"][i]) * upto[-1]).sum()), vocab - 1))
        pad = [-1] * (width - len(path))
        keep.append(path + pad), kept.append(len(path)), tokens.append(said + pad)
        at += t
    return [_int32(keep), _int32(kept), _int32(tokens)]


def exact(case, seed):
    kind = case["kind"]
    lens, counts = _sizes(case)
    if kind in ("attend", "weigh") and sum(n + t for n, t in zip(lens, counts)) * case["kv"] * case["dim"] > 1 << 29:
        return None
    s = _inputs(case, seed)
    if kind == "store":
        return [_exact_e2m1(x) for x in s["new"]]
    if kind == "verify":
        return _exact_verify(s, case)
    if kind == "attend":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
        last, v = None, None
        for i, at, pos, h, g, z in _exact_attention(s, case):
            if last != (i, h):
                last, v = (i, h), _exact_head(s["v"], s["table"][i], pos, h, case)
            lse[at:at + z.shape[0], g] = torch.logsumexp(z, dim=1)
            out[at:at + z.shape[0], g] = torch.softmax(z, dim=1) @ v
        return [out, lse]
    if kind == "weigh":
        mass = s["mass"].double()
        for i, at, pos, _, g, z in _exact_attention(s, case):
            mass[i, :pos.numel()] += torch.exp(z - s["lse"][at:at + z.shape[0], g].double()[:, None]).sum(dim=0)
        return mass
    keep = torch.full((case["seqs"], case["budget"]), -1, dtype=torch.int32)
    new = torch.zeros(s["mass"].shape, dtype=torch.float64)
    for i, n in enumerate(s["host"]):
        mass = s["mass"][i].double().cpu().numpy()
        sinks, recent = min(case["sinks"], n), max(n - case["recent"], 0)
        if n <= case["budget"]:
            rows = np.arange(n)
        else:
            middle = np.arange(sinks, max(recent, sinks))
            best = middle[np.lexsort((middle, -mass[middle]))][:case["budget"] - sinks - (n - max(recent, sinks))]
            rows = np.sort(np.concatenate([np.arange(sinks), best, np.arange(max(recent, sinks), n)]))
        keep[i, :len(rows)] = torch.from_numpy(rows.astype(np.int32))
        new[i, :len(rows)] = torch.from_numpy(mass[rows])
    return [keep.cuda(), torch.minimum(s["lens"], _int32(case["budget"])), new.cuda()]

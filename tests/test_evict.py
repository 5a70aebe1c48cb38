"""The attention weight that cached rows get, and the rows that stay, against the
definition in float64.

Tolerance of the weights. With u = 2^-24, s = scale q . K_r and test_cache.py's error of a
score, dim u scale sum |q K_r| + 4 u |s|: a term exp(s - lse) is off by that much relative,
4 u |lse| for lse times log2 e, 4 u |s - lse| for the fused multiply and add and 4 u for exp2 and the
factor; a sum of n of them, in any order, by n u of it, and adding it to what was gathered by
2 u of both. Rows that stay are equal: the choice compares inputs, and rounds nothing.
"""

import ctypes

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_BF16, cache
from test_cache import TYPES, U, attend, check, make, on, plain
from test_cache4 import call_args, decode, encode, in_4_bits, page_bytes
from test_cache_arguments import as_device, no_launch  # noqa: F401


def plain_lse(c, scale=None):
    """What attention leaves, [nodes, heads] in 32 bits, -inf where a node sees nothing."""
    return torch.from_numpy(walk(c, None, None, scale)[2]).float()


def walk(c, lse, counted, scale=None):
    """Weight of every position, its bound, and each node's log sum, in float64."""
    q, k = c["q"].double().numpy(), c["k"].double().numpy()
    mask, table, cu = c["mask"].numpy().view(np.uint64), c["table"].numpy(), c["cu"].tolist()
    nodes, heads, dim = q.shape
    pages, page, kv = k.shape[:3]
    scale = dim ** -0.5 if scale is None else scale
    lens = c["lens"].tolist()
    cols = max(n + cu[s + 1] - cu[s] for s, n in enumerate(lens))
    got, tol, logs = np.zeros((len(lens), cols)), np.zeros((len(lens), cols)), np.full((nodes, heads), -np.inf)
    for s, n in enumerate(lens):
        for i in range(cu[s], cu[s + 1]):
            t = cu[s + 1] - cu[s]
            pos = [r for r in range(n + t)
                   if r < n or (r - n) // 64 < mask.shape[1] and int(mask[i, (r - n) // 64]) >> ((r - n) % 64) & 1]
            pos = np.array([r for r in pos if r // page < table.shape[1] and 0 <= table[s, r // page] < pages], dtype=int)
            factor = 1.0 if counted is None else float(counted[i])
            if not len(pos) or factor == 0:
                continue
            kr = k[table[s, pos // page], pos % page]
            for h in range(heads):
                kh = kr[:, h * kv // heads]
                z = kh @ q[i, h] * scale
                logs[i, h] = z.max() + np.log(np.exp(z - z.max()).sum())
                if lse is None or float(lse[i, h]) == -np.inf:
                    continue
                at = float(lse[i, h])
                p = np.exp(z - at) * factor
                d = dim * U * scale * (np.abs(kh) @ np.abs(q[i, h])) + 4 * U * (np.abs(z) + abs(at) + np.abs(z - at) + 1)
                got[s, pos] += p
                tol[s, pos] += np.abs(p) * d
    return got, tol + (max(cu[s + 1] - cu[s] for s in range(len(lens))) * heads + 2) * U * np.abs(got), logs


def weigh(d, lse, mass, **kw):
    return cache.row_weights(d["q"], d["k"], d["table"], d["lens"], d["cu"], d["mask"], lse, mass, max_len=d["max_len"],
                             max_tree=d["max_tree"], **kw)


def check_weights(c, d, cuda, lse=None, counted=None, scale=None, extra=5):
    """c: the values that the cache holds, d: the call's tensors on the device."""
    lse = plain_lse(c, scale) if lse is None else lse
    want, tol, _ = walk(c, lse, counted, scale)
    seqs, cols = want.shape
    start = torch.rand((seqs, cols + extra), generator=torch.Generator().manual_seed(1))
    mass = start.to(cuda)
    kw = {} if scale is None else dict(scale=scale)
    got = weigh(d, lse.to(cuda), mass, counted=None if counted is None else counted.to(cuda), **kw)
    assert got is mass
    got, before = got.cpu().double().numpy(), start.double().numpy()
    assert np.array_equal(got[:, cols:], before[:, cols:])
    bound = tol + 2 * U * (np.abs(before[:, :cols]) + np.abs(want))
    assert (np.abs(got[:, :cols] - before[:, :cols] - want) <= bound).all()
    untouched = want == 0
    assert np.array_equal(got[:, :cols][untouched], before[:, :cols][untouched])
    return mass


# ---- refusals (no device needed) --------------------------------------------------

P, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)


@pytest.mark.parametrize("four", [False, True])
def test_weights_refusals(spiral_lib, four):
    d = dict(type=TYPE_BF16, q=P, qn=256, qh=64, nodes=3, heads=4, k=P, pages=8, page=16, kv=2, dim=64, ps=2048)
    d.update({} if four else dict(rs=128, hs=64))
    d.update(table=P, ts=4, cols=4, lens=P, cu=P, seqs=2, mask=P, words=1, max_len=40, max_tree=2, scale=0.125, lse=P,
             counted=P, mass=P, ms=50, mc=50, stream=None)
    fn = spiral_lib.spiral_cache4_row_weights if four else spiral_lib.spiral_cache_row_weights

    def call(**over):
        return fn(*call_args(d, over))

    assert call(type=0) == 6
    for bad in (dict(heads=3), dict(dim=12), dict(dim=264), dict(page=0), dict(pages=0), dict(ts=3), dict(words=-1),
                dict(max_tree=-1), dict(max_len=-1), dict(scale=0.0), dict(scale=float("nan")), dict(mc=-1), dict(ms=49),
                dict(seqs=65536), dict(qn=-8), *([dict(dim=48), dict(page=8), dict(ps=1072)] if four else [dict(rs=-8)])):
        assert call(**bad) == 1, bad
    for bad in (dict(qn=4), dict(q=ODD), dict(k=ODD), dict(mask=ODD), dict(lse=ODD), dict(counted=ODD), dict(mass=ODD),
                dict(cu=ODD), *([] if four else [dict(rs=12), dict(ps=2052), dict(hs=4)])):
        assert call(**bad) == 2, bad
    for bad in (dict(q=None), dict(k=None), dict(table=None), dict(lens=None), dict(cu=None), dict(mask=None),
                dict(lse=None), dict(mass=None)):
        assert call(**bad) == 3, bad
    assert call(nodes=0) == 0 and call(seqs=0) == 0 and call(max_tree=0) == 0 and call(mc=0, ms=0) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert call() == 4 and call(counted=None) == 4


def test_evict_refusals(spiral_lib):
    d = dict(mass=P, ms=100, mc=100, lens=P, seqs=2, budget=20, sinks=4, recent=10, keep=P, ks=20, kept=P,
             new=ctypes.c_void_p(8192), ns=100, ws=None, wsb=0, stream=None)

    def call(**over):
        return spiral_lib.spiral_cache_evict(*call_args(d, over))

    for bad in (dict(ms=99), dict(mc=-1), dict(seqs=-1), dict(seqs=65536), dict(budget=-1), dict(sinks=-1), dict(recent=-1),
                dict(sinks=11), dict(sinks=21, recent=0), dict(recent=1 << 62), dict(ks=19), dict(ns=99), dict(new=P),
                dict(mc=1 << 31, ms=1 << 31)):
        assert call(**bad) == 1, bad
    for bad in (dict(mass=ODD), dict(lens=ODD), dict(keep=ODD), dict(kept=ODD), dict(new=ODD)):
        assert call(**bad) == 2, bad
    for bad in (dict(mass=None), dict(lens=None), dict(keep=None), dict(kept=None)):
        assert call(**bad) == 3, bad
    assert call(ws=ODD) == 2 and call(seqs=0) == 0
    size = spiral_lib.spiral_cache_evict_workspace_bytes
    assert size(8192, 2) == size(1 << 30, 2) == size(65536, 0) == size(65536, 60000) == size(-1, 3) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert call() == 4 and call(new=None) == 4


def test_wrapper_refusals(no_launch):  # noqa: F811
    c = make([5, 6], [2, 2], 2, 1, 64, 16, torch.bfloat16)
    c = {n: as_device(t) if torch.is_tensor(t) else t for n, t in c.items()}
    lse, mass = as_device(torch.zeros(4, 2)), as_device(torch.zeros(2, 9))
    for bad, what in ((dict(lse=as_device(torch.zeros(4, 3))), "lse"), (dict(lse=torch.zeros(4, 2)), "device"),
                      (dict(mass=as_device(torch.zeros(3, 9))), "mass"), (dict(mass=as_device(torch.zeros(1, 9).expand(2, -1))), "overlap"),
                      (dict(counted=as_device(torch.zeros(3))), "counted")):
        kw = {"lse": lse, "mass": mass, **bad}
        with pytest.raises(ValueError, match=what):
            weigh(c, kw.pop("lse"), kw.pop("mass"), **kw)
    with pytest.raises(ValueError, match="the same"):
        weigh({**c, "k": as_device(c["k"].half())}, lse, mass)
    with pytest.raises(ValueError, match="too few words"):
        weigh({**c, "max_tree": 65}, lse, mass)
    with pytest.raises(ValueError, match="mass"):
        cache.evict(torch.zeros(2, 9), c["lens"], 4)
    with pytest.raises(ValueError, match="lens"):
        cache.evict(mass, as_device(c["lens"].long()), 4)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(mass, c["lens"], -1)


# ---- weights ------------------------------------------------------------------------------


CASES = [  # lens, trees, heads, cached heads, dim, page
    ([1], [1], 1, 1, 32, 16), ([0], [3], 4, 2, 64, 16), ([31, 0, 33, 16], [1, 2, 0, 3], 4, 4, 128, 16),
    ([700, 3], [1, 5], 8, 1, 128, 48), ([130, 0, 400], [17, 64, 4], 12, 6, 64, 32), ([300, 45], [25, 7], 6, 3, 96, 16),
    ([200, 90], [30, 12], 5, 1, 160, 16), ([260], [9], 8, 8, 192, 16), ([600, 20], [64, 2], 8, 1, 256, 16),
    ([150], [130], 10, 10, 64, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("case", CASES, ids=[f"{c[2]}x{c[3]}x{c[4]}" for c in CASES])
def test_weights(cuda, case, dtype, four):
    lens, trees, heads, kv, dim, page = case
    c = make(lens, trees, heads, kv, dim, page, dtype, seed=dim + heads)
    call, held = in_4_bits(c) if four else (c, c)
    check_weights(held, on(call, cuda), cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 8, 136, 248])
def test_weights_of_other_dims(cuda, dim):
    c = make([77, 5], [3, 20], 4, 2, dim, 7, torch.float16, seed=dim)
    check_weights(c, on(c, cuda), cuda)


SMALL = [(False, d) for d in (8, 16, 24, 40, 72, 96, 136, 160, 200, 232)] + [(True, d) for d in (32, 96, 160, 192, 224)]


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("four,dim", SMALL)
def test_what_lies_next_to_a_query(cuda, four, dim, many):
    """Queries among NaN, behind them in their rows, in the heads and the nodes beside them, and in
    nodes that are left out: none of it reaches a weight. Both forms, of few and of many queries."""
    lens, trees = ([500 + 2 * i for i in range(64)], [9] * 64) if many else ([77, 5], [3, 20])
    c = make(lens, trees, 8 if many else 4, 2, dim, 16 if four else 7, torch.bfloat16, seed=dim)
    call, held = in_4_bits(c) if four else (c, c)
    nodes, heads, _ = c["q"].shape
    counted = torch.ones(nodes)
    counted[1::2] = 0.0
    lse = plain_lse(held)
    c["q"][1::2], lse[1::2] = float("nan"), float("nan")
    d = on({**call, "q": c["q"]}, cuda)
    wide = torch.full((nodes + 2, heads + 2, dim + 8), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[1:-1, 1:-1, :dim] = d["q"]
    check_weights(held, {**d, "q": wide[1:-1, 1:-1, :dim]}, cuda, lse=lse, counted=counted)
    if many:
        return
    tight = torch.full((nodes + 2, heads, dim), float("nan"), dtype=torch.bfloat16, device=cuda)
    tight[1:-1] = d["q"]
    check_weights(held, {**d, "q": tight[1:-1]}, cuda, lse=lse, counted=counted)


@pytest.mark.gpu
@pytest.mark.parametrize("four,dim", SMALL)
def test_infinities_in_a_query(cuda, four, dim):
    """Scores of minus and plus infinity are weights of 0 and infinity: dims past the head's
    have no part in them."""
    c = make([50], [4], 4, 2, dim, 16, torch.bfloat16, seed=dim, kind="chain")
    c["k"][..., 0] = torch.where(torch.arange(16)[:, None] < 8, 1.0, -1.0).to(torch.bfloat16)
    call, held = in_4_bits(c) if four else (c, c)
    lse = plain_lse(held)
    c["q"][2, 1, 0] = float("inf")
    mass = weigh(on({**call, "q": c["q"]}, cuda), lse.to(cuda), torch.zeros((1, 54), device=cuda))[0].cpu()
    assert torch.equal(mass == float("inf"), (torch.arange(54) % 16 < 8) & (torch.arange(54) < 53))
    assert torch.isfinite(mass[mass != float("inf")]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("heads,kv,dim", [(40, 2, 64), (33, 1, 128), (64, 1, 96), (17, 1, 256), (51, 3, 32)])
def test_more_queries_a_head_than_a_tile(cuda, four, heads, kv, dim):
    c = make([900, 33], [3, 7], heads, kv, dim, 16, torch.bfloat16, seed=heads)
    call, held = in_4_bits(c) if four else (c, c)
    d = on(call, cuda)
    check(attend(d), plain(held))
    check_weights(held, d, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("max_len", [0, 100, 1 << 29])
def test_lengths_that_max_len_does_not_say(cuda, four, max_len):
    """It decides the grid alone: attention and weights of longer and of far shorter rows."""
    c = make([1500, 0, 700], [20, 3, 1], 8, 2, 64, 16, torch.bfloat16, seed=8)
    call, held = in_4_bits(c) if four else (c, c)
    d = on({**call, "max_len": max_len}, cuda)
    check(attend(d), plain(held))
    check_weights(held, d, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_no_sequences_and_no_nodes(cuda, four):
    c = make([40, 3], [2, 1], 4, 2, 64, 16, torch.bfloat16, seed=8)
    d = on(in_4_bits(c)[0] if four else c, cuda)
    none = {**d, "q": d["q"][:0], "mask": d["mask"][:0], "cu": torch.zeros_like(d["cu"])}
    empty = {**none, "table": d["table"][:0], "lens": d["lens"][:0], "cu": d["cu"][:1]}
    for e, seqs in ((none, 2), (empty, 0)):
        out, lse = attend(e)
        mass = torch.rand((seqs, 50), device=cuda)
        before = mass.clone()
        assert out.shape == (0, 4, 64) and torch.equal(weigh(e, lse, mass), before)
        keep, kept, new = cache.evict(mass, e["lens"], 10, sinks=1, recent=2)
        assert keep.shape == (seqs, 10) and kept.tolist() == [10, 3][:seqs] and new.shape == mass.shape
    keep, kept, new = cache.evict(torch.empty((2, 0), device=cuda), d["lens"], 4)
    assert (keep == -1).all() and kept.tolist() == [0, 0] and new.shape == (2, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_many_rows_and_queries(cuda, four):
    """Enough rows for the form that holds more of them, ragged, in pages of 48 rows."""
    lens, trees = [900 + 13 * i % 700 for i in range(64)], [1 + 5 * i % 19 for i in range(64)]
    c = make(lens, trees, 8, 2, 64, 48, torch.bfloat16, seed=5)
    call, held = in_4_bits(c) if four else (c, c)
    d = on(call, cuda)
    first = check_weights(held, d, cuda)
    assert torch.equal(first, check_weights(held, d, cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [96, 160, 192, 256])
@pytest.mark.parametrize("four", [False, True])
def test_many_rows_of_other_dims(cuda, dim, four):
    lens, trees = [500 + 37 * i % 300 for i in range(70)], [9 + i % 5 for i in range(70)]
    c = make(lens, trees, 8, 2, dim, 16, torch.float16, seed=dim)
    call, held = in_4_bits(c) if four else (c, c)
    check_weights(held, on(call, cuda), cuda)


@pytest.mark.gpu
def test_weights_sum_to_the_queries(cuda):
    """With attention's own lse every query of every head gives one."""
    c = make([3000, 100], [9, 2], 8, 2, 128, 16, torch.bfloat16, seed=4)
    d = on(c, cuda)
    _, lse = cache.tree_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], d["cu"], d["mask"], max_len=d["max_len"],
                                  max_tree=d["max_tree"])
    mass = weigh(d, lse, torch.zeros((2, 3009), device=cuda))
    got = mass.double().sum(1).cpu().numpy()
    # Off by test_cache's bound of lse, 128 u scale sum |q K| and the count of rows, relative.
    assert np.abs(got / (8 * np.array([9, 2])) - 1).max() < 2e-3


@pytest.mark.gpu
@pytest.mark.parametrize("four", [False, True])
def test_factors_masks_and_holes(cuda, four):
    """Nodes that are left out whatever they hold, nodes that see nothing, pages that are not there."""
    c = make([50, 200, 0], [6, 3, 4], 4, 2, 128, 16, torch.bfloat16, seed=7, kind="random")
    c["table"][1, 3] = -1
    c["table"][1, 5] = 10 ** 7
    call, held = in_4_bits(c) if four else (c, c)
    counted = torch.tensor([1, 0, 0.5, 0, 2, 1, 1, 0, 1, 1, 0, 1, 0.25])
    lse = plain_lse(held)
    lse[8], lse[1] = -float("inf"), float("nan")
    call, held = dict(call), dict(held)
    q = c["q"].clone()
    q[3], q[7] = float("nan"), float("inf")
    call["q"] = held["q"] = q
    check_weights(held, on(call, cuda), cuda, lse=lse, counted=counted, scale=0.2)


@pytest.mark.gpu
def test_hidden_rows_have_no_weight(cuda):
    """Keys of NaN in rows that are past the end, without a page, or not seen."""
    c = make([20], [5], 2, 1, 64, 16, torch.float16, seed=3, kind="empty")
    c["k"][c["table"][0, 1], 6] = float("nan")  # position 22, a node that none sees
    check_weights(c, on(c, cuda), cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["empty", "chain"])
def test_factors_that_are_nan(cuda, kind):
    """A factor of NaN reaches the rows that its node sees, and no others."""
    c = make([0, 40], [9, 4], 2, 1, 64, 16, torch.bfloat16, seed=6, kind=kind)
    counted = torch.ones(13)
    counted[4] = counted[12] = float("nan")
    mass = weigh(on(c, cuda), plain_lse(c).to(cuda), torch.zeros((2, 44), device=cuda), counted=counted.to(cuda)).isnan().cpu()
    seen = torch.zeros((2, 44), dtype=torch.bool)
    for s, node, n, t in ((0, 4, 0, 9), (1, 12, 40, 4)):
        seen[s, :n] = True
        for j in range(t):
            seen[s, n + j] = bool(int(c["mask"][node, 0]) >> j & 1)
    assert torch.equal(mass, seen)


@pytest.mark.gpu
def test_narrow_mass(cuda):
    """Positions past the columns are left out; rows of a wider buffer and pages far apart."""
    c = make([100, 40], [4, 4], 4, 2, 64, 16, torch.bfloat16, seed=1)
    lse = plain_lse(c)
    want, tol, _ = walk(c, lse, None)
    wide = torch.zeros((2, 300), device=cuda)
    d = on(c, cuda)
    far = torch.full((d["k"].size(0), 2, 16, 2, 64), float("nan"), dtype=torch.bfloat16, device=cuda)
    far[:, 0] = d["k"]
    d["k"] = far[:, 0]
    got = weigh(d, lse.to(cuda), wide[:, 7:60])
    assert (wide[:, :7] == 0).all() and (wide[:, 60:] == 0).all()
    assert (np.abs(got.cpu().double().numpy() - want[:, :53]) <= tol[:, :53]).all()


# ---- rows that stay ------------------------------------------------------------------------


def chosen(mass, n, budget, sinks, recent):
    n = min(max(n, 0), len(mass))
    if n <= budget:
        return np.arange(n)
    value = np.where(np.isnan(mass[:n]), np.inf, mass[:n].astype(np.float64))
    above = np.isnan(mass[:n])
    middle = np.arange(sinks, n - recent)
    order = np.lexsort((middle, -value[middle], ~above[middle]))  # NaN, then by weight, then by place
    best = middle[order[:budget - sinks - recent]]
    return np.sort(np.concatenate([np.arange(sinks), best, np.arange(n - recent, n)]))


def check_evict(mass, lens, budget, sinks, recent, cuda, **kw):
    m = torch.from_numpy(mass).to(cuda)
    keep, kept, new = cache.evict(m, torch.tensor(lens, dtype=torch.int32, device=cuda), budget, sinks=sinks, recent=recent, **kw)
    assert keep.shape == (len(lens), budget) and new.shape == m.shape and np.array_equal(m.cpu().numpy(), mass, equal_nan=True)
    for s, n in enumerate(lens):
        rows = chosen(mass[s], n, budget, sinks, recent)
        assert int(kept[s]) == len(rows)
        assert keep[s].tolist() == rows.tolist() + [-1] * (budget - len(rows))
        assert np.array_equal(new[s].cpu().numpy(), np.concatenate([mass[s][rows], np.zeros(mass.shape[1] - len(rows), dtype=np.float32)]),
                              equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("cols,budget,sinks,recent", [
    (1, 0, 0, 0), (1, 1, 0, 0), (5, 3, 1, 1), (100, 64, 0, 0), (1000, 10, 4, 6), (1025, 300, 4, 100), (4096, 4095, 0, 1),
    (5000, 1, 0, 0), (5000, 1, 1, 0), (5000, 777, 0, 776), (70001, 20000, 16, 1000), (300000, 2, 1, 0)])
def test_rows_that_stay(cuda, cols, budget, sinks, recent):
    rng = np.random.default_rng(cols)
    lens = [cols, cols // 2, budget, min(budget + 1, cols), 0, -3, cols + 100]
    mass = np.exp(3 * rng.standard_normal((len(lens), cols))).astype(np.float32)
    check_evict(mass, lens, budget, sinks, recent, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [700, 20000])
def test_masses_inside_wider_rows_on_two_streams(cuda, cols):
    """Rows at odd addresses with NaN beside them, two calls at the same time."""
    rng = np.random.default_rng(cols)
    lens, streams, held = [cols, cols - 100, 1], [torch.cuda.Stream() for _ in range(2)], []
    for i in range(2):
        mass = rng.random((3, cols)).astype(np.float32)
        wide = torch.full((3, cols + 9), float("nan"), device=cuda)
        wide[:, 5:5 + cols] = torch.from_numpy(mass).to(cuda)
        held.append((mass, wide[:, 5:5 + cols], torch.tensor(lens, dtype=torch.int32, device=cuda)))
    torch.cuda.synchronize()
    got = []
    for s, (_, m, n) in zip(streams, held):
        with torch.cuda.stream(s):
            got.append(cache.evict(m, n, 333, sinks=2, recent=30))
    torch.cuda.synchronize()
    for (mass, _, _), (keep, kept, new) in zip(held, got):
        for s, n in enumerate(lens):
            rows = chosen(mass[s], n, 333, 2, 30)
            assert keep[s, :int(kept[s])].tolist() == rows.tolist()
            assert np.array_equal(new[s].cpu().numpy(), np.concatenate([mass[s][rows], np.zeros(cols - len(rows), dtype=np.float32)]))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zeros", "few values", "one above", "specials", "negative", "close"])
def test_equal_and_odd_weights(cuda, kind):
    for budget in (1, 50, 3500, 6999):
        check_evict(odd_weights(kind, 7000), [7000, 6500, 3000], budget, min(3, budget), 0, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zeros", "few values", "one above", "specials", "negative", "close"])
def test_equal_and_odd_weights_of_divided_rows(cuda, kind):
    """Over workgroups, which the choice does not depend on: the same with a workspace as without."""
    for cols in (8193, 20000, 140001):
        mass = odd_weights(kind, cols)
        for budget in (1, 5001, cols - 1):
            for ws in (None, torch.empty(16, dtype=torch.uint8, device=cuda)):
                check_evict(mass, [cols, cols - 4000, 16385], budget, min(3, budget), budget // 5, cuda, workspace=ws)


@pytest.mark.gpu
def test_divided_rows_in_a_graph(cuda):
    mass, lens = torch.rand((5, 30000), device=cuda), torch.tensor([30000, 9000, 0, 25000, 2001], dtype=torch.int32, device=cuda)
    ws = cache.evict_workspace(mass)
    cache.evict(mass, lens, 2000, sinks=1, recent=9, workspace=ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = cache.evict(mass, lens, 2000, sinks=1, recent=9, workspace=ws)
    for _ in range(4):
        mass.uniform_()
        want = [t.clone() for t in cache.evict(mass, lens, 2000, sinks=1, recent=9, workspace=ws)]
        ws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))


def odd_weights(kind, cols):
    rng = np.random.default_rng(3)
    mass = np.zeros((3, cols), dtype=np.float32)
    if kind == "few values":
        mass = rng.integers(0, 4, (3, cols)).astype(np.float32)
    elif kind == "one above":
        mass[:, 5000] = 1e-40
    elif kind == "specials":
        mass = rng.choice(np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 1.0, 2.0 ** -149], dtype=np.float32), (3, cols))
        mass[0, ::2] = -np.float32(np.nan)
    elif kind == "negative":
        mass = rng.standard_normal((3, cols)).astype(np.float32)
    elif kind == "close":
        mass = (np.float32(1).view(np.int32) + rng.integers(0, 9, (3, cols))).astype(np.int32).view(np.float32)
    return mass


@pytest.mark.gpu
def test_evicted_and_compacted_in_a_graph(cuda):
    """Weights, choice and compaction captured together, replayed over other queries."""
    c = make([400, 90], [2, 3], 4, 2, 64, 16, torch.bfloat16, seed=2)
    d = on(c, cuda)
    start, mass0 = (d["k"].clone(), d["v"].clone()), torch.rand((2, 410), device=cuda)
    mass, zeros = mass0.clone(), torch.zeros(2, dtype=torch.int32, device=cuda)
    ws = cache.tree_attention_workspace(d["q"], d["k"], 2, d["max_len"], d["max_tree"])

    def step():
        _, lse = cache.tree_attention(d["q"], d["k"], d["v"], d["table"], d["lens"], d["cu"], d["mask"],
                                      max_len=d["max_len"], max_tree=d["max_tree"], workspace=ws)
        weigh(d, lse, mass)
        keep, kept, new = cache.evict(mass, d["lens"], 100, sinks=2, recent=8)
        return keep, kept, new, cache.compact(d["k"], d["v"], d["table"], zeros, keep, kept)

    def reset():
        mass.copy_(mass0)
        d["k"].copy_(start[0])
        d["v"].copy_(start[1])

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        d["q"].normal_()
        reset()
        want = [t.clone() for t in (*step(), mass, d["k"], d["v"])]
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip((*held, mass, d["k"], d["v"]), want))

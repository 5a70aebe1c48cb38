"""The paged cache: tree attention against float64, page copies and compaction
against the same moves on the host, the pool of page ids.

Tolerance of attention. With u = 2^-24 and a query's scores s_r = scale q . K_r
(fp32 sums of exact products): a score is off by at most dim u scale sum |q K_r|
and 4 u |s_r| (the scale and its factor log2 e, the fused multiply and add), so p_r
by that much relative, plus 8 u for exp2 and the factors between maxima. Call the
largest of these over the rows d, rows n, half a step of the type h. Then out =
sum p_r V_r / sum p_r is off by at most (2 d + h + (n + 16) u) sum p_r |V_r| / sum
p_r before its own rounding h |out|; F16 holds p below 2^-14 to 2^-25 absolute, of a
sum of at least 1: 2^-25 sum |V_r| more. lse is off by d + n u + 4 u |lse|.
"""

import ctypes

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_BF16, cache, ops

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16]


def make(lens, counts, heads, kv, dim, page, dtype, seed=0, words=None, spare=3, kind="random"):
    """Inputs of a call on the CPU; every row that no sequence owns is NaN."""
    gen, rng = torch.Generator().manual_seed(seed), np.random.default_rng(seed)
    need = [-(-(n + t) // page) for n, t in zip(lens, counts)]
    total = sum(need) + spare
    order = rng.permutation(total)
    table = np.full((len(lens), max(need + [1])), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = order[at:at + c]
        at += c
    k = torch.full((total, page, kv, dim), float("nan")).to(dtype)
    v = k.clone()
    for s, (n, t) in enumerate(zip(lens, counts)):
        for p in range(need[s]):
            rows = min(page, n + t - p * page)
            k[table[s, p], :rows] = torch.randn((rows, kv, dim), generator=gen).to(dtype)
            v[table[s, p], :rows] = torch.randn((rows, kv, dim), generator=gen).to(dtype)
    nodes = sum(counts)
    q = (1.5 * torch.randn((nodes, heads, dim), generator=gen)).to(dtype)
    words = -(-max(counts + [1]) // 64) if words is None else words
    seen = np.zeros((nodes, 64 * words), dtype=bool)
    at = 0
    for t in counts:
        for i in range(t):
            if kind == "random" and i:
                seen[at + i] = seen[at + rng.integers(0, i)]
            elif kind == "chain" and i:
                seen[at + i] = seen[at + i - 1]
            seen[at + i, i] = kind != "empty"
        at += t
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return dict(q=q, k=k, v=v, table=torch.from_numpy(table), lens=torch.tensor(lens, dtype=torch.int32),
                cu=torch.from_numpy(cu), mask=pack(seen), max_len=max(n + t for n, t in zip(lens, counts)),
                max_tree=max(counts))


def pack(seen):
    bits = seen.reshape(seen.shape[0], -1, 64).astype(np.uint64) << np.arange(64, dtype=np.uint64)
    return torch.from_numpy(np.bitwise_or.reduce(bits, axis=2).view(np.int64))


def plain(c, scale=None):
    """out, lse and their bounds in float64, from the definition."""
    q, k, v = c["q"].double().numpy(), c["k"].double().numpy(), c["v"].double().numpy()
    mask, table, cu = c["mask"].numpy().view(np.uint64), c["table"].numpy(), c["cu"].tolist()
    nodes, heads, dim = q.shape
    pages, page, kv = k.shape[:3]
    scale = dim ** -0.5 if scale is None else scale
    half = torch.finfo(c["q"].dtype).eps / 2
    out, lse = np.zeros((nodes, heads, dim)), np.full((nodes, heads), -np.inf)
    tol, ltol = np.zeros(out.shape), np.zeros(lse.shape)
    for s, n in enumerate(c["lens"].tolist()):
        for i in range(cu[s], cu[s + 1]):
            t = cu[s + 1] - cu[s]
            pos = [r for r in range(n + t)
                   if r < n or (r - n) // 64 < mask.shape[1] and int(mask[i, (r - n) // 64]) >> ((r - n) % 64) & 1]
            pos = [r for r in pos if r // page < table.shape[1] and 0 <= table[s, r // page] < pages]
            if not pos:
                continue
            pos = np.array(pos)
            kr, vr = k[table[s, pos // page], pos % page], v[table[s, pos // page], pos % page]
            for h in range(heads):
                kh, vh = kr[:, h * kv // heads], vr[:, h * kv // heads]
                z = kh @ q[i, h] * scale
                m = z.max()
                p = np.exp(z - m)
                total = p.sum()
                out[i, h] = p @ vh / total
                lse[i, h] = m + np.log(total)
                d = (dim * U * abs(scale) * (np.abs(kh) @ np.abs(q[i, h])) + 4 * U * np.abs(z) + 8 * U).max()
                tol[i, h] = (2 * d + half + (pos.size + 16) * U) * (p @ np.abs(vh) / total) + half * np.abs(out[i, h])
                if c["q"].dtype == torch.float16:
                    tol[i, h] += 2.0 ** -25 * np.abs(vh).sum(axis=0) + 2.0 ** -25
                ltol[i, h] = d + pos.size * U + 4 * U * abs(lse[i, h])
    return out, lse, tol, ltol


def on(c, dev):
    return {n: t.to(dev) if torch.is_tensor(t) else t for n, t in c.items()}


def attend(c, **kw):
    return cache.tree_attention(c["q"], c["k"], c["v"], c["table"], c["lens"], c["cu"], c["mask"],
                                max_len=c["max_len"], max_tree=c["max_tree"], **kw)


def check(got, want):
    (out, lse), (wo, wl, tol, ltol) = got, want
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    assert np.array_equal(np.isneginf(lse), np.isneginf(wl))
    some = np.isfinite(wl)
    assert (np.abs(lse[some] - wl[some]) <= ltol[some]).all()
    assert (np.abs(out - wo) <= tol).all(), np.nanmax(np.abs(out - wo) - tol)


# ---- refusals (no device needed) --------------------------------------------------


def tree_args(**over):
    p = ctypes.c_void_p(4096)
    a = dict(type=TYPE_BF16, q=p, qn=256, qh=64, nodes=3, heads=4, k=p, v=p, pages=8, page=16, kv=2, dim=64,
             ps=2048, rs=128, hs=64, table=p, ts=4, cols=4, lens=p, cu=p, seqs=2, mask=p, words=1, max_len=40,
             max_tree=2, scale=0.125, out=p, lse=p, ws=None, wsb=0, stream=None)
    assert not set(over) - set(a)
    a.update(over)
    return list(a.values())


def test_tree_refusals(spiral_lib):
    call = spiral_lib.spiral_tree_attention
    odd = ctypes.c_void_p(4098)
    assert call(*tree_args(type=0)) == 6
    for bad in (dict(heads=3), dict(kv=0), dict(dim=0), dict(dim=12), dict(dim=264), dict(page=0), dict(pages=0),
                dict(pages=1 << 31), dict(cols=-1), dict(ts=3), dict(words=-1), dict(nodes=-1), dict(seqs=65536),
                dict(max_len=-1), dict(max_tree=-1), dict(scale=float("nan")), dict(scale=0.0), dict(rs=-8), dict(ps=1 << 41),
                dict(pages=1 << 30, ps=64), dict(heads=0)):
        assert call(*tree_args(**bad)) == 1, bad
    for bad in (dict(qn=4), dict(rs=12), dict(q=odd), dict(k=odd), dict(v=odd), dict(out=odd), dict(mask=odd),
                dict(table=odd), dict(lens=odd), dict(cu=odd), dict(lse=odd), dict(ws=odd)):
        assert call(*tree_args(**bad)) == 2, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(cu=None),
                dict(mask=None), dict(out=None)):
        assert call(*tree_args(**bad)) == 3, bad
    for none in (dict(nodes=0), dict(seqs=0), dict(max_tree=0)):
        assert call(*tree_args(**none)) == 0, none
    size = spiral_lib.spiral_tree_attention_workspace_bytes
    assert size(4, 3, 64, 2, 4000, 2) == 0 and size(4, 2, 64, 2, 32, 2) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert call(*tree_args()) == 4
        assert call(*tree_args(lse=None, mask=None, words=0)) == 4


def test_move_refusals(spiral_lib):
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
    copy, compact = spiral_lib.spiral_cache_copy_pages, spiral_lib.spiral_cache_compact

    def c(k=p, v=p, layers=2, ls=65536, pages=8, ps=4096, pb=4096, src=p, dst=p, n=3):
        return copy(k, v, layers, ls, pages, ps, pb, src, dst, n, None)

    for bad in (dict(layers=-1), dict(pages=-1), dict(n=-1), dict(pb=0), dict(pb=4100), dict(ps=4000), dict(ls=8),
                dict(layers=40000), dict(n=1 << 40), dict(ls=1 << 61, layers=8)):
        assert c(**bad) == 1, bad
    assert c(k=None) == 3 and c(src=None) == 3 and c(dst=None) == 3
    assert c(k=odd) == 2 and c(v=odd) == 2 and c(src=odd) == 2 and c(dst=odd) == 2
    assert c(n=0) == 0 and c(layers=0) == 0 and c(pages=0) == 0

    def m(k=p, v=p, layers=2, ls=65536, pages=8, ps=4096, page=16, rb=256, table=p, ts=4, cols=4, lens=p, seqs=2,
          keep=p, ks=5, kc=5, kept=p, new=p):
        return compact(k, v, layers, ls, pages, ps, page, rb, table, ts, cols, lens, seqs, keep, ks, kc, kept, new, None)

    for bad in (dict(page=0), dict(rb=0), dict(rb=24), dict(page=17), dict(ps=100), dict(seqs=-1), dict(seqs=65536),
                dict(ts=3), dict(ks=4), dict(kc=-1), dict(pages=-1), dict(layers=-1), dict(rb=1 << 40)):
        assert m(**bad) == 1, bad
    assert m(k=None) == 3 and m(table=None) == 3 and m(lens=None) == 3 and m(keep=None) == 3 and m(kept=None) == 3
    assert m(k=odd) == 2 and m(lens=odd) == 2 and m(new=odd) == 2
    assert m(seqs=0) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert c() == 4 and c(v=None) == 4 and m() == 4 and m(v=None, new=None) == 4 and m(keep=None, kc=0) == 4


def test_wrapper_refusals():
    c = make([5], [2], 2, 1, 16, 4, torch.bfloat16)
    with pytest.raises(ValueError, match="device tensors"):
        attend(c)
    with pytest.raises(ValueError, match="device tensors"):
        cache.copy_pages(c["k"], c["v"], c["lens"], c["lens"])
    with pytest.raises(ValueError, match="device tensors"):
        cache.compact(c["k"], c["v"], c["table"], c["lens"], c["table"], c["lens"])


def test_page_pool():
    pool = cache.PagePool(6, 4)
    a = pool.extend([], 9)
    assert len(a) == 3 and len(set(a)) == 3 and pool.free_pages == 3
    assert pool.extend(a, 12) == a
    b, src, dst = pool.fork(a, 9)
    assert b[:2] == a[:2] and src == [a[2]] and dst == b[2:] and b[2] not in a and pool.free_pages == 2
    d, src, dst = pool.fork(a, 8)
    assert d == a[:2] and src == [] and dst == []
    with pytest.raises(MemoryError):
        pool.alloc(3)
    assert pool.free_pages == 2
    pool.release(a)
    assert pool.free_pages == 3  # the first two pages are still shared
    pool.release(b)
    pool.release(d)
    assert pool.free_pages == 6
    with pytest.raises(ValueError):
        pool.release(a[:1])
    with pytest.raises(ValueError):
        pool.fork(a, 13)
    with pytest.raises(ValueError):
        pool.fork(a, 4)  # released pages
    assert pool.free_pages == 6
    with pytest.raises(ValueError):
        cache.PagePool(4, 0)


# ---- attention ----------------------------------------------------------------------

SHAPES = [
    # lens, trees, heads, kv, dim, page
    ([0], [1], 1, 1, 8, 1),
    ([1], [1], 4, 4, 64, 16),
    ([37], [1], 8, 2, 128, 16),
    ([700], [1], 7, 1, 128, 32),
    ([33, 0, 100], [5, 1, 3], 4, 2, 80, 7),
    ([64, 31], [32, 33], 2, 2, 96, 8),
    ([130, 5, 0, 61], [7, 20, 40, 3], 10, 2, 128, 33),
    ([300, 17], [25, 9], 8, 1, 64, 16),
    ([257], [64], 3, 1, 64, 64),
    ([95, 200], [64, 50], 8, 4, 40, 256),
    ([500, 3], [30, 64], 8, 1, 256, 16),
    ([40], [17], 5, 5, 200, 5),
    ([90], [3], 2, 1, 256, 128),
    ([10, 20], [150, 70], 4, 2, 72, 16),
    ([0], [200], 12, 2, 128, 16),
    ([77], [7], 4, 1, 128, 16),
    ([61], [5], 6, 1, 96, 8),
    ([45, 9], [16, 2], 2, 1, 64, 16),
    ([100], [10], 3, 1, 200, 16),
    ([100, 70], [20, 11], 3, 1, 256, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,trees,heads,kv,dim,page", SHAPES)
def test_tree_attention(cuda, lens, trees, heads, kv, dim, page, dtype):
    c = make(lens, trees, heads, kv, dim, page, dtype, seed=dim + page)
    check(attend(on(c, cuda)), plain(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,trees,heads,kv,dim,page", [
    ([5000], [1], 8, 2, 128, 16), ([3000, 900, 1], [13, 4, 9], 4, 1, 64, 32), ([2000], [40], 4, 2, 128, 64),
    ([2500, 40], [3, 60], 4, 1, 256, 8)])
def test_rows_split_over_workgroups(cuda, lens, trees, heads, kv, dim, page, dtype):
    """The rows of one call split, split less by a smaller workspace, and unsplit."""
    c = make(lens, trees, heads, kv, dim, page, dtype, seed=7)
    want = plain(c)
    d = on(c, cuda)
    full = cache.tree_attention_workspace(d["q"], d["k"], len(lens), d["max_len"], d["max_tree"])
    assert full is not None
    full.fill_(0xFF)
    check(attend(d, workspace=full), want)
    check(attend(d, workspace=full[:full.numel() // 3 // 16 * 16]), want)
    check(attend(d, workspace=full[:16]), want)
    again = [t.clone() for t in attend(d, workspace=full)]
    assert all(torch.equal(a, b) for a, b in zip(again, attend(d, workspace=full)))
    d["max_len"] = 100  # far too low: slower, the same rows
    check(attend(d), want)


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,longest,trees,heads,kv,dim", [
    (70, 900, 3, 4, 1, 64), (130, 300, 9, 8, 2, 128), (513, 150, 1, 2, 2, 64), (5, 2500, 12, 3, 1, 200)])
def test_many_ragged_sequences(cuda, seqs, longest, trees, heads, kv, dim):
    """More sequences than lanes, and than are dealt out; some empty."""
    rng = np.random.default_rng(seqs)
    lens = [int(n) if rng.random() < 0.9 else 0 for n in rng.integers(0, longest, seqs)]
    lens[seqs // 2] = longest
    counts = [int(t) for t in rng.integers(0, trees + 1, seqs)]
    counts[0] = trees
    c = make(lens, counts, heads, kv, dim, 16, torch.float16, seed=seqs)
    check(attend(on(c, cuda)), plain(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["chain", "empty", "random"])
def test_masks(cuda, kind, dtype):
    """Chains, nodes that see no node (with nothing cached: no row at all), masks
    of more words than the trees need, bits of nodes behind one's own."""
    for lens in ([0, 40], [0, 0]):
        c = make(lens, [40, 3], 4, 2, 64, 16, dtype, seed=3, kind=kind, words=2)
        if kind == "random":
            c["mask"][2] = -1  # every bit, past the tree's end too
        check(attend(on(c, cuda)), plain(c))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_infinities_and_nan_where_masked(cuda, bad, dim, dtype):
    """Rows that a node does not see leave no trace in it; those that see them get
    what the sum gives."""
    c = make([70, 20], [20, 8], 8, 2, dim, 16, dtype, seed=5)
    want = plain(c)
    pos, pages = 70 + 13, c["table"]
    for t in ("k", "v"):
        c[t][pages[0, pos // 16], pos % 16] = bad if t == "v" else 0.5
    c["k"][pages[1, 25 // 16], 25 % 16, :, ::3] = bad
    sees = (c["mask"][:20, 0] >> 13 & 1).bool().numpy()
    sees_k = (c["mask"][20:, 0] >> 5 & 1).bool().numpy()
    out, lse = attend(on(c, cuda))
    free = np.concatenate([~sees, ~sees_k])
    check((out[torch.from_numpy(free)], lse[torch.from_numpy(free)]), [t[free] for t in want])
    hit = out[:20].double().cpu().numpy()[sees]
    assert np.isnan(hit).all() if np.isnan(bad) else (hit == bad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_that_are_not_there(cuda, dtype):
    """Negative and too large page ids and a table that ends early hide their rows."""
    c = make([200, 90], [6, 3], 4, 2, 64, 16, dtype, seed=8)
    c["table"][0, 2] = -1
    c["table"][0, 5] = c["k"].size(0)
    c["table"][1, 0] = 2 ** 31 - 1
    c["table"][1, 5] = -2 ** 31
    check(attend(on(c, cuda)), plain(c))
    c["table"] = c["table"][:, :4].contiguous()
    check(attend(on(c, cuda)), plain(c))
    c["table"] = torch.full_like(c["table"], -7)
    out, lse = attend(on(c, cuda))
    assert not out.any() and torch.isneginf(lse).all()


@pytest.mark.gpu
def test_lengths_that_do_not_fit(cuda):
    """Negative and huge lengths, offsets past the nodes: no fault, and the other
    sequence as it was."""
    c = make([40, 30], [4, 4], 2, 1, 64, 16, torch.bfloat16, seed=1)
    want = plain(c)
    d = on(c, cuda)
    for lens, cu in (([-5, 30], [0, 4, 8]), ([2 ** 31 - 1, 30], [0, 4, 8]), ([40, 30], [-3, 4, 1 << 20]),
                     ([40, 30], [0, 4, 2])):
        d["lens"] = torch.tensor(lens, dtype=torch.int32, device=cuda)
        d["cu"] = torch.tensor(cu, dtype=torch.int32, device=cuda)
        out, lse = attend(d)
        torch.cuda.synchronize()
        if cu[1:] == [4, 8]:
            check((out[4:], lse[4:]), [t[4:] for t in want])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 184])
def test_strides(cuda, dim, dtype):
    """Queries out of a fused projection, keys and values out of one buffer with
    heads in front of rows, a table out of a wider one, a given scale, no lse."""
    c = make([77, 3], [9, 2], 6, 2, dim, 16, dtype, seed=2)
    want = plain(c, scale=0.21)
    d = on(c, cuda)
    fused = torch.full((11, 10, dim), float("nan"), dtype=dtype, device=cuda)
    fused[:, 2:8] = d["q"]
    both = torch.full((d["k"].size(0), 2, 2, 16, dim + 8), float("nan"), dtype=dtype, device=cuda)
    both[:, 0, ..., :dim] = d["k"].transpose(1, 2)
    both[:, 1, ..., :dim] = d["v"].transpose(1, 2)
    wide = torch.full((2, d["table"].size(1) + 5), -1, dtype=torch.int32, device=cuda)
    wide[:, 2:2 + d["table"].size(1)] = d["table"]
    d["q"], d["table"] = fused[:, 2:8], wide[:, 2:2 + d["table"].size(1)]
    d["k"], d["v"] = (both[:, i, ..., :dim].transpose(1, 2) for i in (0, 1))
    out, lse = torch.empty_like(c["q"], device=cuda), torch.empty((11, 6), device=cuda)
    got = attend(d, scale=0.21, out=out, lse=lse)
    assert got[0] is out and got[1] is lse
    check(got, want)


@pytest.mark.gpu
def test_wrapper_refuses_on_device(cuda):
    d = on(make([40], [4], 4, 2, 64, 16, torch.bfloat16), cuda)
    for change, match in ((dict(q=d["q"].float()), "bfloat16"), (dict(k=d["k"].half()), "bfloat16"),
                          (dict(v=d["v"][1:]), "layout"), (dict(lens=d["lens"].long()), "lens"),
                          (dict(mask=d["mask"].int()), "mask"), (dict(cu=d["cu"][:1]), "table needs"),
                          (dict(q=d["q"][..., :32]), "one dim"), (dict(max_tree=65), "too few words")):
        with pytest.raises(ValueError, match=match):
            attend({**d, **change})


@pytest.mark.gpu
def test_far_rows(cuda):
    """A cache of more than 2^32 bytes and 2^31 elements: pages at its far end."""
    page, kv, dim = 256, 8, 128
    pages = (1 << 32) // (page * kv * dim * 2) + 5000
    k = torch.empty((pages, page, kv, dim), dtype=torch.bfloat16, device=cuda)
    v = torch.empty_like(k)
    c = make([300], [5], 8, 8, dim, page, torch.bfloat16, seed=4)
    d = on(c, cuda)
    far = [pages - 1, pages // 2 + 3]
    for i, p in enumerate(far):
        k[p], v[p] = d["k"][c["table"][0, i]], d["v"][c["table"][0, i]]
    d.update(k=k, v=v, table=torch.tensor([far], dtype=torch.int32, device=cuda))
    check(attend(d), plain(c))
    ids = lambda *a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    cache.copy_pages(k, v, ids(pages - 1), ids(1))
    assert torch.equal(k[1].view(torch.int16), k[pages - 1].view(torch.int16))
    table = ids(pages - 2, pages - 1)[None]
    k[pages - 2] = 1.0
    k[pages - 1] = 2.0
    assert cache.compact(k, v, table, ids(250), ids(3, 9)[None], ids(2)).tolist() == [252]
    assert (k[pages - 2, :251] == 1).all() and (k[pages - 2, 251] == 2).all() and (k[pages - 2, 252:] == 1).all()


# ---- copies and compaction ------------------------------------------------------------


def bits_of(shape, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return torch.randint(-2 ** 15, 2 ** 15, shape, generator=gen, dtype=torch.int16).view(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("layers,pages,page,kv,dim,n", [
    (1, 5, 1, 1, 8, 2), (3, 9, 16, 2, 64, 4), (2, 40, 8, 8, 128, 17), (48, 7, 3, 1, 24, 3), (1, 300, 16, 4, 128, 140)])
def test_copy_pages(cuda, layers, pages, page, kv, dim, n):
    k, v = (bits_of((layers, pages, page, kv, dim), torch.bfloat16, s) for s in (1, 2))
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).int()
    src, dst = order[:n].clone(), order[n:2 * n].clone()
    if n > 2:
        src[1], dst[2] = -1, pages  # pairs that are left out
    kd, vd = k.to(cuda), v.to(cuda)
    cache.copy_pages(kd, vd, src.to(cuda), dst.to(cuda))
    for s, d in zip(src.tolist(), dst.tolist()):
        if 0 <= s < pages and 0 <= d < pages:
            k[:, d], v[:, d] = k[:, s], v[:, s]
    assert torch.equal(kd.cpu().view(torch.int16), k.view(torch.int16))
    assert torch.equal(vd.cpu().view(torch.int16), v.view(torch.int16))
    cache.copy_pages(kd, vd, src[:0].to(cuda), dst[:0].to(cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("layers,lens,rows,kept,page,kv,dim", [
    (1, [0], 1, [1], 1, 1, 8),
    (2, [5, 0, 33], 20, [7, 0, 20], 16, 2, 64),
    (1, [1000], 4000, [3000], 16, 1, 8),
    (1, [13], 2500, [1200], 64, 8, 128),
    (4, [3, 700, 64, 1], 300, [150, 299, 300, 1], 7, 4, 128),
    (48, [17], 40, [11], 32, 1, 80),
])
@pytest.mark.parametrize("with_values", [True, False])
def test_compact(cuda, layers, lens, rows, kept, page, kv, dim, with_values):
    rng = np.random.default_rng(rows)
    need = [-(-(n + rows) // page) for n in lens]
    total = sum(need) + 2
    order = rng.permutation(total).astype(np.int32)
    table = np.full((len(lens), max(need)), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = order[at:at + c]
        at += c
    keep = np.full((len(lens), max(kept + [1]) + 2), -9, dtype=np.int32)
    for s, c in enumerate(kept):
        keep[s, :c] = np.sort(rng.choice(rows, c, replace=False))
    shape = (layers, total, page, kv, dim)
    caches = [bits_of(shape, torch.float16, s) for s in ((1, 2) if with_values else (1,))]
    dev = [t.to(cuda) for t in caches]
    new = cache.compact(dev[0], dev[1] if with_values else None, torch.from_numpy(table).to(cuda),
                        torch.tensor(lens, dtype=torch.int32, device=cuda), torch.from_numpy(keep).to(cuda),
                        torch.tensor(kept, dtype=torch.int32, device=cuda))
    assert new.tolist() == [a + b for a, b in zip(lens, kept)]
    for got, t in zip(dev, caches):
        t = t.view(torch.int16)
        for s, n in enumerate(lens):
            f, j = n + keep[s, :kept[s]], n + np.arange(kept[s])
            t[:, table[s, j // page], j % page] = t[:, table[s, f // page], f % page].clone()
        assert torch.equal(got.cpu().view(torch.int16), t)


@pytest.mark.gpu
def test_compact_clips(cuda):
    """Counts out of range, rows past the table or on missing pages: left out."""
    k = bits_of((1, 6, 4, 1, 8), torch.float16, 1)
    ids = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda)  # noqa: E731
    table = ids([[0, 1], [2, -1], [3, 99]])
    d = k.to(cuda)
    new = cache.compact(d, None, table, ids([2, 1, 0]), ids([[1, 3, 700], [2, 5, 6], [1, 4, 5]]), ids([9, 3, -4]))
    assert new.tolist() == [5, 4, 0]
    t = k.view(torch.int16)
    t[0, 0, 2], t[0, 0, 3] = t[0, 0, 3].clone(), t[0, 1, 1].clone()
    t[0, 2, 1] = t[0, 2, 3].clone()
    assert torch.equal(d.cpu().view(torch.int16), t)
    with pytest.raises(ValueError, match="pages contiguous"):
        cache.compact(d.transpose(2, 4), None, table, ids([0, 0, 0]), ids([[0]] * 3), ids([0, 0, 0]))


# ---- together -------------------------------------------------------------------------


@pytest.mark.gpu
def test_captured_and_on_another_stream(cuda):
    """Attention, a page copy and compaction in one graph, replayed on new contents
    with eager calls in between."""
    c = make([600, 90], [12, 30], 8, 2, 128, 16, torch.bfloat16, seed=6)
    d = on(c, cuda)
    ws = cache.tree_attention_workspace(d["q"], d["k"], 2, d["max_len"], d["max_tree"])
    spare = torch.tensor([i for i in range(d["k"].size(0)) if i not in c["table"].flatten().tolist()][:1],
                         dtype=torch.int32, device=cuda)
    keep = torch.tensor([[0, 2, 5, 11], [1, 3, 4, 29]], dtype=torch.int32, device=cuda)
    kept = torch.tensor([4, 3], dtype=torch.int32, device=cuda)
    out, lse = torch.empty_like(d["q"]), torch.empty((42, 8), device=cuda)
    page = d["table"][0, :1].contiguous()

    def call(k, v, o, z):
        cache.tree_attention(d["q"], k, v, d["table"], d["lens"], d["cu"], d["mask"], max_len=d["max_len"],
                             max_tree=d["max_tree"], out=o, lse=z, workspace=ws)
        cache.copy_pages(k, v, page, spare)
        return cache.compact(k, v, d["table"], d["lens"], keep, kept)

    side = torch.cuda.Stream()
    k0, v0 = d["k"].nan_to_num(), d["v"].nan_to_num()
    k, v = k0.clone(), v0.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(k, v, out, lse)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new = call(k, v, out, lse)
    for i in range(4):
        a, b = k0 * (1 + 0.25 * i), v0.flip(-1) * (1 + i)
        k.copy_(a)
        v.copy_(b)
        out.fill_(float("nan"))
        graph.replay()
        got = [t.clone() for t in (out, lse, k, v, new)]
        want = [a, b, torch.empty_like(out), torch.empty_like(lse)]
        lens = call(*want)
        torch.cuda.synchronize()
        for x, y in zip(got, [want[2], want[3], a, b, lens]):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_one_node_is_plain_decoding(cuda):
    """A tree of one node against torch's attention over the same rows in float64."""
    c = make([1234], [1], 8, 2, 128, 16, torch.float16, seed=9)
    out, _ = attend(on(c, cuda))
    pos = torch.arange(1235)
    k, v = (c[t][c["table"][0, pos // 16].long(), pos % 16].double().repeat_interleave(4, dim=1) for t in ("k", "v"))
    p = torch.softmax((c["q"][0].double()[None] * k).sum(-1) * 128 ** -0.5, dim=0)
    want = (p[..., None] * v).sum(0)
    _, _, tol, _ = plain(c)
    assert ((out[0].double().cpu() - want).abs().numpy() <= tol[0]).all()


@pytest.mark.gpu
def test_quantized_projection_into_the_cache(cuda):
    """Keys from an MXFP4 product written to the cache, then read by attention: the
    calls share torch's stream."""
    gen = torch.Generator().manual_seed(1)
    w = ops.mxfp4_quantize((torch.randn((128, 256), generator=gen) / 16).bfloat16().to(cuda))
    x = torch.randn((20, 256), generator=gen).bfloat16().to(cuda)
    rows = ops.mul_mat(39, w, 128, 256, x).view(20, 2, 64)
    c = make([16], [4], 2, 2, 64, 10, torch.bfloat16, seed=1)
    d = on(c, cuda)
    d["k"][d["table"][0].long()] = rows.view(2, 10, 2, 64)
    got = attend(d)
    c["k"] = d["k"].cpu()
    check(got, plain(c))

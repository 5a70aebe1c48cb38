"""The cache in 4 bits: rows stored against an encoder in float64, bytes and all; read
back, moved and copied; tree attention against float64 over the values that the codes
stand for.

Tolerance of attention: test_cache.py's. The codes are exact in both 16-bit types, so its
terms for the scores, the softmax, P's rounding to 16 bits and the output's hold as they
stand.
"""

import ctypes

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_BF16, cache
from test_cache import TYPES, attend, check, make, on, plain
from test_cache_arguments import as_device, no_launch  # noqa: F401

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
FLOATS = [torch.float32, torch.float16, torch.bfloat16]


# ---- the format on the host --------------------------------------------------------


def encode(x):
    """Codes [..., dim] and scale bytes [..., dim / 32] of float64 rows."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    odd = ~np.isfinite(b).all(-1, keepdims=True)
    b = np.where(odd, 0.0, b)
    top = np.abs(b).max(-1, keepdims=True)
    e = np.clip(np.frexp(top)[1] - 3, -127, 127)
    e = np.where(top == 0, -127, e)
    a = np.abs(b) * 2.0 ** -e.astype(np.float64)
    code = np.zeros(a.shape, dtype=np.uint8)
    for c in range(7):  # ties go to the even code
        border = (E2M1[c] + E2M1[c + 1]) / 2
        code += (a >= border) if c % 2 else (a > border)
    code = np.where(odd, 0, code + 8 * np.signbit(b).astype(np.uint8))
    return code.reshape(x.shape).astype(np.uint8), np.where(odd, 255, e + 127)[..., 0].astype(np.uint8)


def decode(code, scale):
    f = np.where(scale == 255, np.nan, 2.0 ** (scale.astype(np.float64) - 127))
    v = E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    return (v.reshape(*v.shape[:-1], -1, 32) * f[..., None]).reshape(v.shape)


def page_bytes(code, scale):
    """Pages [pages, page, kv, dim] of codes and their scales as the cache holds them."""
    pages, page, kv, dim = code.shape
    pair = (code[..., 0::2] | code[..., 1::2] << 4).transpose(0, 2, 1, 3).reshape(pages, kv, -1)
    return torch.from_numpy(np.concatenate([pair, scale.transpose(0, 2, 3, 1).reshape(pages, kv, -1)], axis=2))


def in_4_bits(c):
    """test_cache's inputs with the cache in 4 bits, and for plain() the values it holds."""
    four, held = dict(c), dict(c)
    for n in ("k", "v"):
        code, scale = encode(c[n].double().numpy())
        four[n], held[n] = page_bytes(code, scale), torch.from_numpy(decode(code, scale))
    return four, held


# ---- refusals (no device needed) --------------------------------------------------


def call_args(defaults, over):
    assert not set(over) - set(defaults)
    return list({**defaults, **over}.values())


P, ODD = ctypes.c_void_p(4096), ctypes.c_void_p(4098)
WHERE = dict(table=P, ts=4, cols=4, lens=P, cu=P, seqs=2)


def test_page_bytes(spiral_lib):
    size = spiral_lib.spiral_cache4_page_bytes
    assert size(16, 8, 128) == 16 * 8 * 4 * 17 and size(48, 1, 32) == 48 * 17
    for bad in ((8, 8, 128), (0, 8, 128), (16, 0, 128), (16, 8, 48), (16, 8, 0), (16, 8, 288), (-16, 8, 128)):
        assert size(*bad) == 0, bad


def test_store_and_load_refusals(spiral_lib):
    d = dict(type=TYPE_BF16, nk=P, nv=P, ns=512, hs=64, nodes=3, k=P, v=P, pages=8, page=16, kv=2, dim=64, ps=1088,
             **WHERE, stream=None)

    def store(**over):
        return spiral_lib.spiral_cache4_store(*call_args(d, over))

    assert store(type=8) == 6
    for bad in (dict(page=8), dict(dim=48), dict(dim=288), dict(kv=0), dict(ps=1072), dict(ps=1096), dict(pages=-1),
                dict(nodes=-1), dict(seqs=-1), dict(seqs=65536), dict(ts=3), dict(cols=-1), dict(ns=-8),
                dict(nodes=1 << 25), dict(page=1 << 24)):
        assert store(**bad) == 1, bad
    for bad in (dict(ns=4), dict(hs=4), dict(nk=ODD), dict(nv=ODD), dict(k=ODD), dict(v=ODD), dict(table=ODD),
                dict(lens=ODD), dict(cu=ODD)):
        assert store(**bad) == 2, bad
    for bad in (dict(nk=None), dict(k=None), dict(nv=None), dict(v=None), dict(table=None), dict(lens=None), dict(cu=None)):
        assert store(**bad) == 3, bad
    for none in (dict(nodes=0), dict(seqs=0), dict(pages=0)):
        assert store(**none) == 0, none
    e = dict(type=TYPE_BF16, k=P, pages=8, page=16, kv=2, dim=64, ps=1088, **WHERE, nodes=3, out=P, stream=None)

    def load(**over):
        return spiral_lib.spiral_cache4_load(*call_args(e, over))

    assert load(type=0) == 6 and load(page=17) == 1 and load(ps=1000) == 1 and load(out=ODD) == 2 and load(k=ODD) == 2
    assert load(k=None) == 3 and load(out=None) == 3 and load(nodes=0) == 0 and load(seqs=0) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert store() == 4 and store(nv=None, v=None) == 4 and store(type=0, ns=4, hs=4) == 4 and load() == 4


def test_attention_refusals(spiral_lib):
    d = dict(type=TYPE_BF16, q=P, qn=256, qh=64, nodes=3, heads=4, k=P, v=P, pages=8, page=16, kv=2, dim=64, ps=1088,
             **WHERE, mask=P, words=1, max_len=40, max_tree=2, scale=0.125, out=P, lse=P, ws=None, wsb=0, stream=None)

    def call(**over):
        return spiral_lib.spiral_cache4_tree_attention(*call_args(d, over))

    assert call(type=0) == 6
    for bad in (dict(heads=3), dict(dim=48), dict(page=8), dict(pages=0), dict(ps=1072), dict(ps=1096), dict(ts=3),
                dict(words=-1), dict(max_tree=-1), dict(scale=0.0), dict(scale=float("inf")), dict(qn=-8),
                dict(cols=1 << 24, ts=1 << 24)):
        assert call(**bad) == 1, bad
    for bad in (dict(qn=4), dict(qh=4), dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(out=ODD), dict(mask=ODD), dict(ws=ODD),
                dict(lse=ODD), dict(cu=ODD)):
        assert call(**bad) == 2, bad
    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(table=None), dict(lens=None), dict(cu=None),
                dict(mask=None), dict(out=None)):
        assert call(**bad) == 3, bad
    assert call(nodes=0) == 0 and call(seqs=0) == 0 and call(max_tree=0) == 0
    size = spiral_lib.spiral_cache4_tree_attention_workspace_bytes
    assert size(4, 2, 48, 2, 4000, 2) == 0 and size(4, 2, 64, 2, 32, 2) == 0
    assert 0 < size(32, 8, 128, 256, 8192, 64) <= 256 << 20
    if spiral_lib.spiral_device_count() == 0:
        assert call() == 4


def test_compact_refusals(spiral_lib):
    d = dict(k=P, v=P, layers=2, ls=65536, pages=8, ps=1088, page=16, kv=2, dim=64, table=P, ts=4, cols=4, lens=P, seqs=2,
             keep=P, ks=5, kc=5, kept=P, new=P, stream=None)

    def call(**over):
        return spiral_lib.spiral_cache4_compact(*call_args(d, over))

    for bad in (dict(page=8), dict(dim=40), dict(ps=1072), dict(layers=-1), dict(ls=8), dict(ls=1 << 61, layers=8),
                dict(seqs=-1), dict(ts=3), dict(ks=4), dict(kc=-1), dict(pages=-1)):
        assert call(**bad) == 1, bad
    assert call(k=None) == 3 and call(table=None) == 3 and call(keep=None) == 3 and call(kept=None) == 3
    assert call(k=ODD) == 2 and call(new=ODD) == 2 and call(seqs=0) == 0
    if spiral_lib.spiral_device_count() == 0:
        assert call() == 4 and call(v=None, new=None) == 4


def test_wrapper_refusals(no_launch):  # noqa: F811
    c, _ = in_4_bits(make([5, 6], [2, 2], 2, 1, 64, 16, torch.bfloat16))
    c = {n: as_device(t) if torch.is_tensor(t) else t for n, t in c.items()}
    new = as_device(torch.zeros(4, 1, 64))
    where = c["table"], c["lens"], c["cu"]
    with pytest.raises(ValueError, match="multiple of 16 rows"):
        attend({**c, "k": as_device(c["k"][..., :-17].contiguous()), "v": as_device(c["v"][..., :-17].contiguous())})
    with pytest.raises(ValueError, match="one layer"):
        attend({**c, "k": c["k"][None], "v": c["v"][None]})
    with pytest.raises(ValueError, match="uint8"):
        attend({**c, "v": as_device(c["v"].float())})
    with pytest.raises(ValueError, match="go together"):
        cache.store4(new, None, c["k"], c["v"], *where)
    with pytest.raises(ValueError, match="heads"):
        cache.store4(as_device(torch.zeros(4, 2, 64)), None, c["k"], None, *where)
    with pytest.raises(ValueError, match="contiguous dim"):
        cache.store4(as_device(torch.zeros(4, 1, 128)[..., ::2]), None, c["k"], None, *where)
    with pytest.raises(ValueError, match="cu an entry"):
        cache.store4(new, None, c["k"], None, c["table"], c["lens"], c["lens"])
    with pytest.raises(ValueError, match="table.*overlap"):
        cache.store4(new, None, c["k"], None, as_device(c["table"][:1].expand(2, -1)), c["lens"], c["cu"])
    with pytest.raises(ValueError, match="out must be"):
        cache.load4(c["k"], *where, new)
    with pytest.raises(ValueError, match="needs dim"):
        cache.compact(c["k"], c["v"], c["table"], c["lens"], c["table"], c["lens"])
    with pytest.raises(ValueError, match="pages contiguous"):
        cache.copy_pages(as_device(c["k"][..., ::2]), None, c["lens"], c["lens"])


def test_empty4_refuses():
    for bad in ((4, 8, 2, 64), (4, 16, 2, 48), (-1, 16, 2, 64), (4, 16, 0, 64)):
        with pytest.raises(ValueError):
            cache.empty4(*bad, device="cpu")
    assert cache.empty4(3, 32, 2, 96, layers=2, device="cpu").shape == (2, 3, 2, 32 * 51)


# ---- rows in and out ----------------------------------------------------------------


def rows_case(lens, counts, kv, dim, page, seed=0):
    """A table with a negative id, one past the pages and too few columns for the last rows."""
    rng = np.random.default_rng(seed)
    need = [-(-(n + t) // page) for n, t in zip(lens, counts)]
    total = sum(need) + 2
    order = rng.permutation(total)
    table = np.full((len(lens), max(need)), -1, dtype=np.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = order[at:at + c]
        at += c
    return table, total, np.concatenate([[0], np.cumsum(counts)]).astype(np.int32), rng


def positions(table, lens, counts, page, total):
    """(node, page id, row) of every node that has a page."""
    at, out = 0, []
    for s, (n, t) in enumerate(zip(lens, counts)):
        for i in range(t):
            p = (n + i) // page
            if p < table.shape[1] and 0 <= table[s, p] < total:
                out.append((at + i, table[s, p], (n + i) % page))
        at += t
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("lens,counts,kv,dim,page", [
    ([0], [1], 1, 32, 16), ([5, 0, 100, 31], [3, 0, 70, 1], 2, 64, 16), ([63, 64, 1], [2, 1, 200], 3, 96, 48),
    ([0] * 70 + [17], [1] * 70 + [40], 8, 128, 16), ([1000], [300], 1, 256, 64), ([7, 8], [9, 10], 5, 160, 32)])
def test_store_and_load(cuda, dtype, lens, counts, kv, dim, page):
    table, total, cu, rng = rows_case(lens, counts, kv, dim, page)
    if table.size > 3:
        table[-1, -1], table[0, 0] = -5, total
    nodes = int(cu[-1])
    x = (rng.standard_normal((2, nodes, kv, dim)) * np.exp2(rng.integers(-6, 7, (2, nodes, kv, 1)))).astype(np.float32)
    x[0, 0, 0, :32] = 0.0  # a block of nothing, of both signs
    x[0, 0, 0, 1] = -0.0
    if nodes > 2:
        x[1, 1, 0, 5], x[0, 1, -1, -1], x[0, 2, 0, 3] = np.nan, np.inf, -np.inf
        x[1, 2, 0, :32] = np.float32(2.0 ** -24) * np.arange(32)  # subnormal in F16
        x[0, nodes - 1, 0, :32] = [0.25 * i - 4 for i in range(32)]  # ties
    # A slice of wider rows, as of a fused projection.
    wide = torch.zeros((nodes, 2 * kv + 3, dim), dtype=dtype)
    wide[:, 1:1 + kv], wide[:, 1 + kv:1 + 2 * kv] = torch.from_numpy(x[0]), torch.from_numpy(x[1])
    d = wide.to(cuda)
    new = d[:, 1:1 + kv], d[:, 1 + kv:1 + 2 * kv]
    start = torch.from_numpy(rng.integers(0, 256, (2, total, kv, page * dim * 17 // 32), dtype=np.uint8))
    caches = [t.to(cuda) for t in start]
    tt, tl, tc = torch.from_numpy(table).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda), torch.from_numpy(cu).to(cuda)
    cache.store4(*new, *caches, tt, tl, tc)
    there = positions(table, lens, counts, page, total)
    for got, src, was in zip(caches, (wide[:, 1:1 + kv], wide[:, 1 + kv:1 + 2 * kv]), start):
        code, scale = encode(src.double().numpy())
        want = was.numpy().copy()
        codes = want[..., :page * dim // 2].reshape(total, kv, page, dim // 2)
        scales = want[..., page * dim // 2:].reshape(total, kv, dim // 32, page)
        for n, p, r in there:
            codes[p, :, r] = code[n, :, 0::2] | code[n, :, 1::2] << 4
            scales[p, :, :, r] = scale[n]
        flat = np.concatenate([codes.reshape(total, kv, -1), scales.reshape(total, kv, -1)], axis=2)
        assert np.array_equal(got.cpu().numpy(), flat)
        held = np.zeros((nodes, kv, dim))
        for n, _, _ in there:
            held[n] = decode(code[n], scale[n])
        for t in TYPES:
            out = torch.full((nodes, kv, dim), 7.0, dtype=t, device=cuda)
            assert cache.load4(got, tt, tl, tc, out) is out
            assert np.array_equal(out.double().cpu().numpy(), torch.from_numpy(held).to(t).double().numpy(), equal_nan=True)
    only = start[0].to(cuda)  # keys alone
    cache.store4(new[0], None, only, None, tt, tl, tc)
    assert torch.equal(only, caches[0])


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_nodes_of_no_sequence(device):
    """Read back as zeros, also where there is no sequence at all."""
    on_device = as_device if device == "cpu" else lambda t: t.cuda()
    k = on_device(torch.full((3, 2, 16 * 34), 0x77, dtype=torch.uint8))
    for seqs in (0, 2) if device == "cuda" else (0,):
        table, lens = on_device(torch.zeros((seqs, 1), dtype=torch.int32)), on_device(torch.zeros(seqs, dtype=torch.int32))
        cu = on_device(torch.tensor([2] * seqs + [2], dtype=torch.int32))
        out = on_device(torch.full((5, 2, 64), 7.0, dtype=torch.bfloat16))
        assert cache.load4(k, table, lens, cu, out) is out and (out == 0).all()


@pytest.mark.gpu
def test_every_code_and_scale(cuda):
    """Each code under each scale byte, read back in both types."""
    code = np.arange(256 * 32).reshape(256, 1, 32) % 16
    scale = np.arange(256, dtype=np.uint8).reshape(256, 1, 1)
    bytes_ = page_bytes(code.reshape(16, 16, 1, 32).astype(np.uint8), scale.reshape(16, 16, 1, 1)).to(cuda)
    table = torch.arange(16, dtype=torch.int32, device=cuda)[None]
    lens, cu = torch.zeros(1, dtype=torch.int32, device=cuda), torch.tensor([0, 256], dtype=torch.int32, device=cuda)
    for t in TYPES:
        out = cache.load4(bytes_, table, lens, cu, torch.empty((256, 1, 32), dtype=t, device=cuda))
        want = torch.from_numpy(decode(code, scale)).to(t).double().numpy()
        assert np.array_equal(out.double().cpu().numpy(), want, equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("layers,kv,dim,page", [(None, 1, 32, 16), (3, 2, 96, 32), (2, 8, 128, 16), (1, 5, 256, 48)])
def test_copies_and_compaction(cuda, layers, kv, dim, page):
    rng = np.random.default_rng(dim)
    lens, most, rows = [0, 37, page, 5], 90, 97
    need = [-(-(n + rows) // page) for n in lens]
    table, total, _, _ = rows_case(lens, [rows] * 4, kv, dim, page, seed=page)
    kept = [90, 0, 41, 1]
    keep = np.full((4, most + 3), -1, dtype=np.int32)
    for s, c in enumerate(kept):
        keep[s, :c] = np.sort(rng.choice(rows, c, replace=False))
    if need[2] > 1:
        table[2, need[2] - 1] = total + 4  # rows without a page stay where they are
    shape = (total, kv, page * dim * 17 // 32) if layers is None else (layers, total, kv, page * dim * 17 // 32)
    start = [rng.integers(0, 256, shape, dtype=np.uint8) for _ in range(2)]
    k, v = (torch.from_numpy(t).to(cuda) for t in start)
    tt, tl = torch.from_numpy(table).to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    new = cache.compact(k, v, tt, tl, torch.from_numpy(keep).to(cuda)[:, :most], torch.tensor(kept, dtype=torch.int32, device=cuda), dim)
    assert new.tolist() == [n + c for n, c in zip(lens, kept)]
    half = page * dim // 2
    for got, want in zip((k, v), start):
        want = want.reshape(-1, total, kv, page * dim * 17 // 32).copy()
        codes, scales = want[..., :half].reshape(-1, total, kv, page, dim // 2).copy(), want[..., half:].reshape(-1, total, kv, dim // 32, page).copy()
        for s, c in enumerate(kept):
            for j in range(c):
                a, b = lens[s] + keep[s, j], lens[s] + j
                pa, pb = table[s, a // page], table[s, b // page]
                if 0 <= pa < total and 0 <= pb < total:
                    codes[:, pb, :, b % page] = codes[:, pa, :, a % page]
                    scales[:, pb, :, :, b % page] = scales[:, pa, :, :, a % page]
        flat = np.concatenate([codes.reshape(-1, total, kv, half), scales.reshape(-1, total, kv, page * dim // 32)], axis=3)
        assert np.array_equal(got.cpu().numpy().reshape(flat.shape), flat)
    before = k.clone(), v.clone()
    src, dst = torch.tensor([3, 1], dtype=torch.int32, device=cuda), torch.tensor([0, 2], dtype=torch.int32, device=cuda)
    cache.copy_pages(k, v, src, dst)
    for got, want in zip((k, v), before):
        want = want.view(-1, total, kv, page * dim * 17 // 32)
        want[:, [0, 2]] = want[:, [3, 1]]
        assert torch.equal(got.view(want.shape), want)


# ---- attention ------------------------------------------------------------------------


CASES = [  # lens, trees, heads, cached heads, dim, page
    ([1], [1], 1, 1, 32, 16),
    ([0], [1], 4, 2, 64, 16),
    ([31, 0, 33, 16, 15], [1, 1, 2, 0, 3], 4, 2, 128, 16),
    ([700, 3, 64], [1, 5, 2], 8, 1, 128, 48),
    ([130, 0, 1000], [17, 64, 4], 8, 2, 64, 32),
    ([300, 45], [25, 7], 6, 2, 96, 16),
    ([500], [40], 16, 2, 128, 64),
    ([200, 90], [30, 12], 5, 1, 160, 16),
    ([260, 1500], [9, 1], 8, 8, 192, 16),
    ([100, 3], [3, 64], 7, 1, 224, 32),
    ([3000, 20], [64, 2], 8, 1, 256, 16),
    ([0, 10], [150, 1], 4, 4, 32, 32),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES, ids=[f"{c[2]}x{c[3]}x{c[4]}" for c in CASES])
def test_attention(cuda, case, dtype):
    lens, trees, heads, kv, dim, page = case
    c = make(lens, trees, heads, kv, dim, page, dtype, seed=dim + heads)
    four, held = in_4_bits(c)
    check(attend(on(four, cuda)), plain(held))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["empty", "chain"])
def test_masks(cuda, kind):
    """Nodes that see nothing, chains of several words, and a sequence without a cached row."""
    c = make([0, 50, 0], [130, 3, 1], 4, 2, 128, 16, torch.bfloat16, seed=3, kind=kind)
    four, held = in_4_bits(c)
    out, lse = attend(on(four, cuda))
    check((out, lse), plain(held))
    if kind == "empty":
        assert torch.isneginf(lse[:130]).all() and (out[:130] == 0).all()


WIDE = [  # from 32 tiles of 16 queries on; chains are prompts in chunks
    ([1000, 40], [150, 3], 8, 2, 128, 16, "random"),
    ([2100], [131], 4, 1, 96, 32, "random"),
    ([90, 0], [600, 520], 1, 1, 64, 16, "chain"),
    ([0, 700], [140, 513], 4, 4, 32, 16, "chain"),
    ([3000, 1], [130, 129], 4, 1, 160, 16, "random"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", WIDE, ids=[f"{c[2]}x{c[3]}x{c[4]}" for c in WIDE])
def test_many_queries(cuda, case, dtype):
    lens, trees, heads, kv, dim, page, kind = case
    c = make(lens, trees, heads, kv, dim, page, dtype, seed=dim, kind=kind)
    four, held = in_4_bits(c)
    d, want = on(four, cuda), plain(held)
    check(attend(d), want)
    check(attend(d, workspace=torch.empty(16, dtype=torch.uint8, device=cuda)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,trees", [(4, 64, [1, 2]), (8, 128, [1, 1]), (16, 128, [20, 9]), (2, 256, [1, 33])])
def test_split_and_workspace(cuda, heads, dim, trees):
    """Long rows over workgroups: with all, some and no workspace, run after run the same."""
    c = make([5000, 700], trees, heads, 2, dim, 16, torch.float16, seed=heads)
    four, held = in_4_bits(c)
    d, want = on(four, cuda), plain(held)
    full = cache.tree_attention_workspace(d["q"], d["k"], 2, d["max_len"], d["max_tree"])
    assert full is not None
    per = heads * (dim * 4 + 8)
    for size in (full.numel(), 5 * per, per, 16):
        ws = full[:size].fill_(0xFF)
        got = [t.clone() for t in attend(d, workspace=ws)]
        check(got, want)
        assert all(torch.equal(a, b) for a, b in zip(got, attend(d, workspace=ws)))


BATCHES = {  # lens, trees, heads, cached heads, dim
    # More sequences than a wave has lanes, some without a tree, waves divided by each tree's queries.
    "ragged": ([97 * i % 1900 for i in range(80)], [(0, 1, 1, 40, 3, 9, 0, 17)[i % 8] for i in range(80)], 8, 2, 64),
    "ragged, wide heads": ([131 * i % 1500 for i in range(70)], [(33, 1, 0, 5)[i % 4] for i in range(70)], 4, 2, 256),
    # A part of all work a place: sequences whole but for the one or two that would end last.
    "one long among many": ([13 * i % 40 for i in range(399)] + [5000], [1 + i % 2 for i in range(400)], 8, 8, 32),
    "a chain, a wide tree among many": ([7 * i % 30 for i in range(150)] + [4000] + [5 * i % 30 for i in range(150)] + [2600, 0],
                                        [1 + i % 3 for i in range(150)] + [1] + [i % 3 for i in range(150)] + [60, 2], 16, 8, 64),
    # One token each, rows for two rounds of workgroups.
    "two rounds": ([311 * i % 2900 for i in range(75)], [1] * 75, 8, 8, 128),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", BATCHES)
def test_batches(cuda, name):
    """Many sequences dealt by their rows and by the time that their trees take, with all, half, little
    and no workspace: every row counted once."""
    lens, trees, heads, kv, dim = BATCHES[name]
    c = make(lens, trees, heads, kv, dim, 16, torch.bfloat16, seed=len(lens))
    four, held = in_4_bits(c)
    d, want = on(four, cuda), plain(held)
    full = cache.tree_attention_workspace(d["q"], d["k"], len(lens), d["max_len"], d["max_tree"])
    assert full is not None
    per = heads * (dim * 4 + 8)
    for lines in (full.numel() // per, full.numel() // per // 2, max(trees) + 3, 0):
        ws = full[:max(lines * per, 16)].fill_(0xFF)
        got = [t.clone() for t in attend(d, workspace=ws)]
        check(got, want)
        assert all(torch.equal(a, b) for a, b in zip(got, attend(d, workspace=ws)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,far", [(torch.bfloat16, 253), (torch.bfloat16, 254), (torch.bfloat16, 255),
                                       (torch.float16, 141), (torch.float16, 142), (torch.float16, 144), (torch.float16, 255)])
@pytest.mark.parametrize("lens,trees", [([40], [6]), ([0], [40]), ([3000], [6])])
def test_values_past_the_type(cuda, dtype, far, lens, trees):
    """V's codes that are infinities or NaN in the type, in rows that some nodes see, none
    do, and all do: as in test_cache's reference over values rounded to the type."""
    c = make(lens, trees, 4, 2, 128, 16, dtype, seed=far + lens[0])
    code, scale = encode(c["v"].double().numpy())
    table = c["table"][0].numpy()
    n = lens[0]
    for row in (n + 1, n + 3) + ((5,) if n and far != 255 else ()):
        scale[table[row // 16], row % 16, :, 1] = far
    kc, ks = encode(c["k"].double().numpy())
    four = dict(c, k=page_bytes(kc, ks), v=page_bytes(code, scale))
    held = dict(c, k=torch.from_numpy(decode(kc, ks)), v=torch.from_numpy(decode(code, scale)).to(dtype).double())
    with np.errstate(invalid="ignore", over="ignore"):
        wo, wl, tol, _ = plain(held)
    out, lse = attend(on(four, cuda))
    out = out.double().cpu().numpy()
    assert np.array_equal(np.isnan(out), np.isnan(wo)) and np.array_equal(np.isposinf(out), np.isposinf(wo))
    assert np.array_equal(np.isneginf(out), np.isneginf(wo))
    big = torch.finfo(dtype).max * 0.9
    some = np.isfinite(wo) & np.isfinite(tol) & (np.abs(wo) < big)
    assert (np.abs(out[some] - wo[some]) <= tol[some]).all()


@pytest.mark.gpu
def test_keys_that_are_nan(cuda):
    """A NaN among the scores makes the node NaN; the same row hidden leaves it as it was."""
    c = make([70], [9], 4, 2, 64, 16, torch.bfloat16, seed=9)
    code, scale = encode(c["k"].double().numpy())
    page = int(c["table"][0, 72 // 16])
    scale[page, 72 % 16, 0, 1] = 255  # node 2's key, head 0
    vc, vs = encode(c["v"].double().numpy())
    four = dict(c, k=page_bytes(code, scale), v=page_bytes(vc, vs))
    out, lse = attend(on(four, cuda))
    sees = (c["mask"][:, 0] >> 2 & 1).bool()
    assert torch.isnan(out.cpu()[:, :2]).all(-1).all(-1).equal(sees) and torch.isnan(lse.cpu()[:, :2]).all(-1).equal(sees)
    assert torch.isfinite(out.cpu()[:, 2:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hole", [-1, 10 ** 6])
def test_pages_that_are_not_there(cuda, hole):
    c = make([300, 20], [3, 2], 4, 2, 128, 16, torch.bfloat16, seed=2)
    c["table"][0, 4], c["table"][0, 7], c["table"][1, 0] = hole, hole, hole
    c["table"] = torch.cat([c["table"], torch.full((2, 2), hole, dtype=torch.int32)], dim=1)
    c["lens"][1] = 21  # rows of page 1 only
    four, held = in_4_bits(c)
    (out, lse), (wo, wl, tol, ltol) = attend(on(four, cuda)), plain(held)
    last = np.isnan(wl[4])  # the second sequence's last node has its row behind those written, which are NaN
    assert last.all() and torch.isnan(lse[4]).all() and torch.isnan(out[4]).all()
    check((out[:4], lse[:4]), (wo[:4], wl[:4], tol[:4], ltol[:4]))


@pytest.mark.gpu
def test_strides_and_streams(cuda):
    """Queries inside wider rows, pages further apart, another stream, given outputs."""
    c = make([100, 37], [5, 1], 4, 2, 96, 16, torch.bfloat16, seed=6)
    four, held = in_4_bits(c)
    d = on(four, cuda)
    wide = torch.full((6, 9, 104), float("nan"), dtype=torch.bfloat16, device=cuda)
    wide[:, 2:6, :96] = d["q"]
    d["q"] = wide[:, 2:6, :96]
    for n in ("k", "v"):
        far = torch.full((d[n].size(0), 3, d[n].size(2)), 0xFF, dtype=torch.uint8, device=cuda)
        far[:, :2] = d[n]
        d[n] = far[:, :2]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty((6, 4, 96), dtype=torch.bfloat16, device=cuda)
        got = attend(d, out=out, scale=0.3)
    side.synchronize()
    assert got[0] is out
    check(got, plain(held, scale=0.3))


@pytest.mark.gpu
def test_pages_past_32_bits(cuda):
    """Pages more than 2^31 bytes apart: every call as over pages side by side."""
    c = make([40, 21], [3, 2], 4, 2, 64, 16, torch.bfloat16, seed=4, spare=0)
    four, held = in_4_bits(c)
    near = on(four, cuda)
    far, (pages, heads, size) = dict(near), near["k"].shape
    step = (1 << 31) + 4096
    for n in ("k", "v"):
        space = torch.empty((pages - 1) * step + heads * size, dtype=torch.uint8, device=cuda)
        far[n] = space.as_strided((pages, heads, size), (step, size, 1))
        far[n].copy_(near[n])
    new = [torch.randn((5, 2, 64), device=cuda) for _ in range(2)]
    keep = torch.tensor([[0, 2], [1, -1]], dtype=torch.int32, device=cuda)
    kept, got = torch.tensor([2, 1], dtype=torch.int32, device=cuda), []
    for d in (near, far):
        cache.store4(*new, d["k"], d["v"], d["table"], d["lens"], d["cu"])
        rows = cache.load4(d["v"], d["table"], d["lens"], d["cu"], new[0].bfloat16())
        out, lse = attend(d)
        mass = cache.row_weights(d["q"], d["k"], d["table"], d["lens"], d["cu"], d["mask"], lse,
                                 torch.zeros((2, 50), device=cuda), max_len=d["max_len"], max_tree=d["max_tree"])
        lens = cache.compact(d["k"], d["v"], d["table"], d["lens"], keep, kept, 64)
        got.append((rows, out, lse, mass, lens, d["k"], d["v"]))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_captured(cuda):
    """Store, attention and compaction in a graph, replayed over new rows."""
    c = make([60, 900], [4, 2], 8, 2, 128, 32, torch.bfloat16, seed=8)
    four, _ = in_4_bits(c)
    d = on(four, cuda)
    start = d["k"].clone(), d["v"].clone()
    new = [torch.empty((6, 2, 128), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
    ws = cache.tree_attention_workspace(d["q"], d["k"], 2, d["max_len"], d["max_tree"])
    keep = torch.tensor([[1, 3], [0, 1]], dtype=torch.int32, device=cuda)
    kept = torch.tensor([2, 1], dtype=torch.int32, device=cuda)

    def step():
        cache.store4(*new, d["k"], d["v"], d["table"], d["lens"], d["cu"])
        out = attend(d, workspace=ws)
        return (*out, cache.compact(d["k"], d["v"], d["table"], d["lens"], keep, kept, 128))

    for t in new:
        t.normal_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        for t in new:
            t.normal_()
        for n, t in zip(("k", "v"), start):
            d[n].copy_(t)
        want = [t.clone() for t in step()] + [d["k"].clone(), d["v"].clone()]
        for n, t in zip(("k", "v"), start):
            d[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*held, d["k"], d["v"]], want))

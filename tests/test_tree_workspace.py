"""The workspace of tree attention, bounded whatever the largest tree is, and what is split
with all, little or none of it: batches of every balance of lengths and trees."""

import numpy as np
import pytest
import torch

from spiral_amd import cache
from test_cache import attend, check, make, on, plain

MOST = 256 << 20


@pytest.mark.parametrize("heads,kv,dim,seqs,max_len,max_tree", [
    (32, 8, 128, 256, 8192, 2048), (64, 8, 128, 512, 8192, 512), (64, 8, 256, 48, 8192, 64),
    (65536, 1, 256, 512, 1 << 29, 1 << 24), (32, 8, 128, 8, 131072, 2048)])
def test_bounded(spiral_lib, heads, kv, dim, seqs, max_len, max_tree):
    """A prompt chunk beside decoding sequences, wide trees, and the largest sizes that the
    call takes (whose tree times group is refused above 2^31)."""
    size = spiral_lib.spiral_tree_attention_workspace_bytes(heads, kv, dim, seqs, max_len, max_tree)
    assert 0 <= size <= MOST


def test_sizes(spiral_lib):
    size = spiral_lib.spiral_tree_attention_workspace_bytes
    assert size(32, 8, 128, 1, 8192, 4096) == 0  # one prompt whose queries fill the GPU
    for seqs, tree in ((1, 1), (16, 25), (48, 1)):  # decoding and drafts: a share for each place, a node for each row
        per = tree * 32 * (128 * 4 + 8)
        n = size(32, 8, 128, seqs, 8192, tree)
        assert n % per == 0 and seqs + 2 <= n // per <= seqs + 512


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("nodes", [1, 30, 4000])
def test_prompt_chunk_beside_decoding(cuda, dim, nodes):
    """One long chunk and single nodes in every order, a workspace of so many nodes in all:
    none, not enough for the chunk, and enough."""
    lens, trees = [900, 1500, 20, 2600, 0, 1400], [150, 1, 1, 2, 0, 1]
    c = make(lens, trees, 8, 2, dim, 16, torch.float16, seed=nodes)
    want = plain(c)
    d = on(c, cuda)
    per = 8 * (dim * 4 + 8)
    ws = torch.full((nodes * per,), 0xFF, dtype=torch.uint8, device=cuda)
    first = [t.clone() for t in attend(d, workspace=ws)]
    check(first, want)
    assert all(torch.equal(a, b) for a, b in zip(first, attend(d, workspace=ws)))
    for order in ([5, 4, 3, 2, 1, 0], [3, 0, 1, 2, 4, 5]):  # the chunk last, the longest first
        first = c["cu"].tolist()
        at = np.concatenate([np.arange(first[s], first[s + 1]) for s in order])
        e = {**c, "q": c["q"][at], "mask": c["mask"][at], "table": c["table"][order], "lens": c["lens"][order],
             "cu": torch.tensor(np.concatenate([[0], np.cumsum([trees[s] for s in order])]), dtype=torch.int32)}
        check(attend(on(e, cuda), workspace=ws), [t[at] for t in want])


BATCHES = {  # lens, trees, heads, cached heads, dim
    "one long among many": ([17 * i % 61 for i in range(199)] + [5000], [1] * 200, 8, 8, 64),
    "a chunk, one long": ([33 * i % 90 for i in range(43)] + [3000, 0], [1 + i % 2 for i in range(44)] + [300], 16, 8, 40),
    "long ones, wide trees": ([1500, 2, 0, 1400, 700], [64, 1, 0, 33, 40], 16, 4, 256),
    "wide rows, one long": ([13 * i % 70 for i in range(99)] + [4000], [1 + i % 3 for i in range(100)], 8, 8, 256),
    "trees of many rows": ([97 * i % 600 for i in range(63)] + [900], [1 + 11 * i % 25 for i in range(63)] + [25], 32, 8, 64),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", BATCHES)
def test_batches(cuda, name):
    """With the workspace that the call allocates, with parts of it and without."""
    lens, trees, heads, kv, dim = BATCHES[name]
    c = make(lens, trees, heads, kv, dim, 16, torch.bfloat16 if dim == 64 else torch.float16, seed=len(lens))
    want, d = plain(c), on(c, cuda)
    full = cache.tree_attention_workspace(d["q"], d["k"], len(lens), d["max_len"], d["max_tree"])
    assert full is not None and full.numel() <= MOST
    check(attend(d), want)
    per = heads * (dim * 4 + 8)
    for lines in (1, 2, 5, 40, 700, full.numel() // per):
        ws = full[:min(lines * per, full.numel())].fill_(0xFF)
        got = [t.clone() for t in attend(d, workspace=ws)]
        check(got, want)
        assert all(torch.equal(a, b) for a, b in zip(got, attend(d, workspace=ws)))

"""A paged key/value cache on the device: attention of drafted trees over it,
page copies for forks, compaction of kept rows (include/spiral_cache.h).

Keys and values are two tensors of one shape and the same strides,
[pages, page, kv_heads, dim] (a layer) or [layers, pages, page, kv_heads, dim],
bfloat16 or float16. A table [seqs, columns] of int32 page ids says where a
sequence's rows lie. Every function launches on torch's current HIP stream and
returns without synchronizing.
"""

from collections import Counter

import torch

from ._lib import TYPE_BF16, TYPE_F16, check, lib

_TYPES = {torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


# The checks below read each property once and put their messages together only when
# they fail: at the smallest calls the host takes longer than the GPU.
def _int32(name, t, dims):
    if t.dtype is torch.int32 and t.is_cuda and t.dim() == dims and (t.stride(-1) == 1 or t.size(-1) <= 1):
        if dims == 1 or t.stride(0) >= t.size(1) or t.size(0) <= 1:
            return
        raise ValueError(f"{name}'s rows overlap (an expanded tensor needs .contiguous())")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a device tensor")
    raise ValueError(f"{name} must be a {dims}-D int32 tensor with contiguous rows")


def tree_attention_workspace(q, k, seqs, max_len, max_tree):
    """Workspace for tree_attention over queries and keys of these shapes, or None
    where it needs none."""
    n = lib().spiral_tree_attention_workspace_bytes(q.size(1), k.size(2), q.size(2), seqs, max_len, max_tree)
    return torch.empty(n, dtype=torch.uint8, device=q.device) if n > 0 else None


def tree_attention(q, k, v, table, lens, cu, mask, *, max_len, max_tree, scale=None, out=None, lse=None,
                   workspace=None):
    """Attention of one tree of drafted tokens per sequence: (out, lse).

    q [nodes, heads, dim]: the nodes of all trees, sequence s's at cu[s] .. cu[s + 1]
    (cu [seqs + 1] int32). k, v [pages, page, kv_heads, dim] hold its lens[s] cached
    rows (lens [seqs] int32) and, behind them, its nodes' own rows. mask [nodes,
    words] int64: bit j of a node's words is set where it sees its tree's node j
    (itself too, as a rule); it sees every cached row. max_len: the longest
    sequence with its tree (decides whether rows are split over workgroups),
    max_tree: no less than the largest tree. scale defaults to dim ** -0.5. out [nodes, heads, dim] in q's
    type, lse [nodes, heads] float32 (natural logarithm of the sum of exponentials;
    -inf and a row of zeros where a node sees nothing). workspace: from
    tree_attention_workspace (allocated here when omitted and needed)."""
    if not (q.is_cuda and k.is_cuda and v.is_cuda and mask.is_cuda):
        raise ValueError("expected device tensors")
    dtype = q.dtype
    kind = _TYPES.get(dtype)
    if kind is None or k.dtype is not dtype or v.dtype is not dtype:
        raise ValueError("q, k and v must be bfloat16 or float16, all the same")
    shape, kshape, sq, sk = q.shape, k.shape, q.stride(), k.stride()
    nodes, heads, dim = shape
    pages, page, kv_heads, kdim = kshape
    if kdim != dim or (dim > 1 and (sq[2] != 1 or sk[3] != 1)):
        raise ValueError("q and k must have one dim, contiguous")
    if v.shape != kshape or v.stride() != sk:
        raise ValueError("keys and values must have one type, shape and layout")
    _int32("table", table, 2)
    _int32("lens", lens, 1)
    _int32("cu", cu, 1)
    seqs = lens.size(0)
    rows, cols = table.shape
    if rows != seqs or cu.size(0) != seqs + 1:
        raise ValueError("table needs a row, cu an entry and one more, for each of lens")
    mask_nodes, words = mask.shape
    if mask.dtype is not torch.int64 or mask_nodes != nodes or not mask.is_contiguous():
        raise ValueError("mask must be a contiguous int64 tensor [nodes, words]")
    if max_tree > 64 * words:
        raise ValueError("mask has too few words for max_tree")
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=q.device)
    elif out.shape != shape or out.dtype is not dtype or not out.is_cuda or not out.is_contiguous():
        raise ValueError("out must be contiguous, on the device, of q's shape and type")
    if lse is None:
        lse = torch.empty((nodes, heads), dtype=torch.float32, device=q.device)
    elif lse.shape != (nodes, heads) or lse.dtype is not torch.float32 or not lse.is_cuda or not lse.is_contiguous():
        raise ValueError("lse must be contiguous float32 [nodes, heads] on the device")
    if workspace is None:
        workspace = tree_attention_workspace(q, k, seqs, max_len, max_tree)
    elif not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be on the device and contiguous")
    ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    check(lib().spiral_tree_attention(
        kind, q.data_ptr(), sq[0], sq[1], nodes, heads, k.data_ptr(), v.data_ptr(), pages, page, kv_heads, dim,
        sk[0], sk[1], sk[2], table.data_ptr(), max(table.stride(0), cols), cols, lens.data_ptr(), cu.data_ptr(), seqs,
        mask.data_ptr(), words, max_len, max_tree, dim ** -0.5 if scale is None else scale, out.data_ptr(),
        lse.data_ptr(), ws, ws_bytes, _stream()), "tree_attention")
    return out, lse


def _layers(k, v):
    """(layers, bytes from layer to layer, pages, from page to page, bytes a page, a row) of a cache."""
    if not k.is_cuda or (v is not None and not v.is_cuda):
        raise ValueError("expected device tensors")
    shape, step, size = k.shape, k.stride(), k.element_size()
    if v is not None and (v.dtype is not k.dtype or v.shape != shape or v.stride() != step):
        raise ValueError("keys and values must have one type, shape and layout")
    if len(shape) == 4:
        shape, step = (1, *shape), (0, *step)
    if len(shape) != 5 or 0 in shape[2:]:
        raise ValueError("a cache is [layers, pages, page, kv_heads, dim] or one layer of it")
    layers, pages, page, heads, dim = shape
    if (dim > 1 and step[4] != 1) or (heads > 1 and step[3] != dim) or (page > 1 and step[2] != heads * dim):
        raise ValueError("a cache needs its pages contiguous")
    row = heads * dim * size
    return layers, step[0] * size, pages, max(step[1] * size, page * row) if pages == 1 else step[1] * size, page * row, row


def copy_pages(k, v, src, dst):
    """Page src[i] over page dst[i] in every layer of k and v (v may be None):
    the copies a fork makes. src, dst int32 [n]; dst distinct and not in src."""
    layers, layer_step, pages, page_step, page_bytes, _ = _layers(k, v)
    _int32("src", src, 1)
    _int32("dst", dst, 1)
    if src.size(0) != dst.size(0):
        raise ValueError("src and dst must be of one length")
    check(lib().spiral_cache_copy_pages(k.data_ptr(), None if v is None else v.data_ptr(), layers, layer_step, pages,
                                        page_step, page_bytes, src.data_ptr(), dst.data_ptr(), src.size(0), _stream()),
          "copy_pages")


def compact(k, v, table, lens, keep, kept):
    """Moves the kept rows of every sequence together, in every layer of k and v (v
    may be None): the row at position lens[s] + keep[s, j] goes to lens[s] + j, for
    j < kept[s]. keep [seqs, most] int32, ascending in each row; table [seqs,
    columns], lens and kept [seqs] int32. Returns the new lengths, lens + kept."""
    layers, layer_step, pages, page_step, page_bytes, row_bytes = _layers(k, v)
    _int32("table", table, 2)
    _int32("lens", lens, 1)
    _int32("keep", keep, 2)
    _int32("kept", kept, 1)
    seqs = lens.size(0)
    if table.size(0) != seqs or keep.size(0) != seqs or kept.size(0) != seqs:
        raise ValueError("table, keep and kept need a row for each of lens")
    new_lens = torch.empty_like(lens)
    check(lib().spiral_cache_compact(k.data_ptr(), None if v is None else v.data_ptr(), layers, layer_step, pages,
                                     page_step, page_bytes // row_bytes, row_bytes, table.data_ptr(),
                                     max(table.stride(0), table.size(1)), table.size(1), lens.data_ptr(), seqs,
                                     keep.data_ptr(), max(keep.stride(0), keep.size(1)), keep.size(1), kept.data_ptr(),
                                     new_lens.data_ptr(), _stream()), "compact")
    return new_lens


class PagePool:
    """Page ids of a cache with reference counts, on the host: what a sequence's
    table row is filled from. Pages are shared between forks until one of them has
    to write, which is the page its last row ends in."""

    def __init__(self, pages, page):
        if pages < 0 or page <= 0:
            raise ValueError("a pool needs pages >= 0 of page > 0 rows")
        self.page = page
        self._refs = [0] * pages
        self._free = list(range(pages - 1, -1, -1))

    @property
    def free_pages(self):
        return len(self._free)

    def alloc(self, n):
        """n page ids, each with one reference; raises MemoryError and takes none
        where fewer are free."""
        if n < 0:
            raise ValueError("n must not be negative")
        if n > len(self._free):
            raise MemoryError(f"{n} pages wanted, {len(self._free)} free")
        ids = [self._free.pop() for _ in range(n)]
        for i in ids:
            self._refs[i] = 1
        return ids

    def extend(self, ids, rows):
        """Page ids of a sequence grown to hold `rows` rows."""
        return list(ids) + self.alloc(max(0, -(-rows // self.page) - len(ids)))

    def fork(self, ids, rows):
        """A second sequence of the first `rows` rows of ids: (its page ids, src,
        dst). Whole pages are shared; the page that row `rows` falls into is the
        fork's own: copy src over dst with copy_pages. Nothing is taken where a page
        is not in use (ValueError) or none is free (MemoryError)."""
        whole, part = divmod(rows, self.page)
        if rows < 0 or whole + (part > 0) > len(ids):
            raise ValueError("ids do not hold that many rows")
        for i in ids[:whole + (part > 0)]:
            self._in_use(i)
        own = self.alloc(1) if part else []
        for i in ids[:whole]:
            self._refs[i] += 1
        return list(ids[:whole]) + own, list(ids[whole:whole + len(own)]), own

    def release(self, ids):
        """Gives back one reference to each page (an id may come as often as it has
        references); those without any become free. Nothing is given back where a page
        is not in use (ValueError)."""
        ids = list(ids)
        for i, n in Counter(ids).items():
            self._in_use(i, n)
        for i in ids:
            self._refs[i] -= 1
            if self._refs[i] == 0:
                self._free.append(i)

    def _in_use(self, i, times=1):
        if not 0 <= i < len(self._refs) or self._refs[i] < times:
            raise ValueError(f"page {i} is not in use" + (f" {times} times" if times > 1 else ""))

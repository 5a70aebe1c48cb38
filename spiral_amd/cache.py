"""A paged key/value cache on the device, in 16 bits or in 4: attention of drafted
trees over it, verification of the drafts, page copies for forks, compaction of kept
rows, eviction by accumulated attention weight (include/spiral_cache.h).

Keys and values are two tensors of one shape and the same strides,
[pages, page, kv_heads, dim] (a layer) or [layers, pages, page, kv_heads, dim],
bfloat16 or float16; or, in MXFP4, uint8 tensors [pages, kv_heads, page * dim * 17 / 32]
or [layers, ...] (empty4), written by store4 and read by everything else as the others
are. A table [seqs, columns] of int32 page ids says where a sequence's rows lie. Every
function launches on torch's current HIP stream and returns without synchronizing.
"""

from collections import Counter

import torch

from ._lib import TYPE_BF16, TYPE_F16, TYPE_F32, check, lib

_TYPES = {torch.bfloat16: TYPE_BF16, torch.float16: TYPE_F16}
_FLOATS = {**_TYPES, torch.float32: TYPE_F32}
_I32, _F32, _U8 = torch.int32, torch.float32, torch.uint8


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


# The checks below read each property once and put their messages together only when
# they fail: at the smallest calls the host takes longer than the GPU.
def _int32(name, t, dims):
    if t.dtype is _I32 and t.is_cuda and t.dim() == dims and t.is_contiguous():
        return
    if t.dtype is torch.int32 and t.is_cuda and t.dim() == dims and (t.stride(-1) == 1 or t.size(-1) <= 1):
        if dims == 1 or t.stride(0) >= t.size(1) or t.size(0) <= 1:
            return
        raise ValueError(f"{name}'s rows overlap (an expanded tensor needs .contiguous())")
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a device tensor")
    raise ValueError(f"{name} must be a {dims}-D int32 tensor with contiguous rows")


def _page4(name, k, dim):
    """Rows a page of a cache in 4 bits, checked."""
    shape, step = k.shape, k.stride()
    if len(shape) not in (3, 4):
        raise ValueError(f"{name}: a cache in 4 bits is [pages, kv_heads, bytes] or [layers, ...]")
    if dim <= 0 or dim > 256 or dim % 32 or shape[-1] <= 0 or shape[-1] % (dim // 32 * 17 * 16):
        raise ValueError(f"{name}: dim must be a multiple of 32 up to 256, a page a multiple of 16 rows of dim * 17 / 32 bytes")
    if not k.is_cuda or k.dtype is not torch.uint8:
        raise ValueError(f"{name}: expected a uint8 device tensor")
    if step[-1] != 1 or (shape[-2] > 1 and step[-2] != shape[-1]):
        raise ValueError(f"{name}: a cache needs its pages contiguous")
    return shape[-1] // (dim // 32 * 17)


def _page_step4(k):
    """Bytes from page to page."""
    shape = k.shape
    return k.stride(-3) if shape[-3] > 1 else shape[-2] * shape[-1]


def empty4(pages, page, kv_heads, dim, layers=None, device="cuda"):
    """Keys (or values) of a cache in 4 bits, all zeros: uint8 [pages, kv_heads, page * dim *
    17 / 32], or [layers, ...]. page: a multiple of 16 rows; dim: of 32, up to 256."""
    n = lib().spiral_cache4_page_bytes(page, kv_heads, dim)
    if n == 0 or pages < 0:
        raise ValueError("a cache in 4 bits needs pages of a multiple of 16 rows, dim a multiple of 32 up to 256")
    shape = (pages, kv_heads, n // kv_heads)
    return torch.zeros(shape if layers is None else (layers, *shape), dtype=torch.uint8, device=device)


def _rows4(table, lens, cu):
    """The arguments that say where rows lie, checked."""
    _int32("table", table, 2)
    _int32("lens", lens, 1)
    _int32("cu", cu, 1)
    seqs, (rows, cols) = len(lens), table.shape
    if rows != seqs or len(cu) != seqs + 1:
        raise ValueError("table needs a row, cu an entry and one more, for each of lens")
    return table.data_ptr(), max(table.stride(0), cols), cols, lens.data_ptr(), cu.data_ptr(), seqs


def store4(new_k, new_v, k, v, table, lens, cu):
    """Rows new_k and new_v [nodes, kv_heads, dim] (float32, float16 or bfloat16, the same
    strides; new_v and v may be None) into a layer of a cache in 4 bits, quantized: node
    cu[s] + i goes to position lens[s] + i of sequence s, behind its cached rows, where
    tree_attention looks for it. Rows without a page are left out."""
    if not new_k.is_cuda or (new_v is not None and not new_v.is_cuda):
        raise ValueError("expected device tensors")
    if (new_v is None) != (v is None):
        raise ValueError("new_v and v go together")
    kind = _FLOATS.get(new_k.dtype)
    nodes, heads, dim = new_k.shape
    step = new_k.stride()
    if kind is None or (new_v is not None and (new_v.dtype is not new_k.dtype or new_v.shape != new_k.shape)):
        raise ValueError("new_k and new_v must be float32, float16 or bfloat16, of one type and shape")
    if dim > 1 and step[2] != 1 or new_v is not None and new_v.stride() != step:
        raise ValueError("new rows need a contiguous dim and the same strides")
    page = _page4("k", k, dim)
    if v is not None and (not v.is_cuda or v.dtype is not _U8 or v.shape != k.shape or v.stride() != k.stride()):
        raise ValueError("keys and values must be on the device, of one type, shape and layout")
    if k.dim() != 3 or k.size(1) != heads:
        raise ValueError("the cache must be one layer with new_k's heads")
    rows = _rows4(table, lens, cu)
    check(lib().spiral_cache4_store(
        kind, new_k.data_ptr(), None if new_v is None else new_v.data_ptr(), step[0], step[1], nodes, k.data_ptr(),
        None if v is None else v.data_ptr(), k.size(0), page, heads, dim, _page_step4(k), *rows, _stream()),
        "store4")


def load4(k, table, lens, cu, out):
    """The rows that store4 would write, read back to out [nodes, kv_heads, dim] (bfloat16 or
    float16, contiguous) as the values they hold; zeros for those without a page."""
    kind = _TYPES.get(out.dtype)
    if kind is None or not out.is_cuda or not out.is_contiguous():
        raise ValueError("out must be contiguous bfloat16 or float16 on the device")
    nodes, heads, dim = out.shape
    page = _page4("k", k, dim)
    if k.dim() != 3 or k.size(1) != heads:
        raise ValueError("the cache must be one layer with out's heads")
    rows = _rows4(table, lens, cu)
    if rows[-1] == 0:  # no sequence has a row
        return out.zero_()
    check(lib().spiral_cache4_load(kind, k.data_ptr(), k.size(0), page, heads, dim, _page_step4(k), *rows, nodes,
                                   out.data_ptr(), _stream()), "load4")
    return out


def tree_attention_workspace(q, k, seqs, max_len, max_tree):
    """Workspace for tree_attention over queries and keys of these shapes, or None
    where it needs none."""
    if k.dtype is torch.uint8:
        n = lib().spiral_cache4_tree_attention_workspace_bytes(q.size(1), k.size(1), q.size(2), seqs, max_len, max_tree)
    else:
        n = lib().spiral_tree_attention_workspace_bytes(q.size(1), k.size(2), q.size(2), seqs, max_len, max_tree)
    return torch.empty(n, dtype=torch.uint8, device=q.device) if n > 0 else None


def tree_attention(q, k, v, table, lens, cu, mask, *, max_len, max_tree, scale=None, out=None, lse=None,
                   workspace=None):
    """Attention of one tree of drafted tokens per sequence: (out, lse).

    q [nodes, heads, dim]: the nodes of all trees, sequence s's at cu[s] .. cu[s + 1]
    (cu [seqs + 1] int32). k, v [pages, page, kv_heads, dim] in q's type, or in 4 bits,
    hold its lens[s] cached rows (lens [seqs] int32) and, behind them, its nodes' own rows. mask [nodes,
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
    four = k.dtype is torch.uint8
    if kind is None or v.dtype is not k.dtype or (k.dtype is not dtype and not four):
        raise ValueError("q, k and v must be bfloat16 or float16, all the same, or k and v uint8 (in 4 bits)")
    shape, kshape, sq, sk = q.shape, k.shape, q.stride(), k.stride()
    nodes, heads, dim = shape
    if dim > 1 and sq[2] != 1:
        raise ValueError("q must have a contiguous dim")
    if four:
        page = _page4("k", k, dim)
        if len(kshape) != 3:
            raise ValueError("tree_attention takes one layer of a cache")
        layout = (kshape[0], page, kshape[1], dim, _page_step4(k))
    else:
        pages, page, kv_heads, kdim = kshape
        if kdim != dim or (dim > 1 and sk[3] != 1):
            raise ValueError("q and k must have one dim, contiguous")
        layout = (pages, page, kv_heads, dim, sk[0], sk[1], sk[2])
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
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype is not dtype or not out.is_cuda or not out.is_contiguous():
        raise ValueError("out must be contiguous, on the device, of q's shape and type")
    if lse is None:
        lse = q.new_empty((nodes, heads), dtype=_F32)
    elif lse.shape != (nodes, heads) or lse.dtype is not torch.float32 or not lse.is_cuda or not lse.is_contiguous():
        raise ValueError("lse must be contiguous float32 [nodes, heads] on the device")
    if workspace is None:
        workspace = tree_attention_workspace(q, k, seqs, max_len, max_tree)
    elif not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be on the device and contiguous")
    ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    call = lib().spiral_cache4_tree_attention if four else lib().spiral_tree_attention
    check(call(
        kind, q.data_ptr(), sq[0], sq[1], nodes, heads, k.data_ptr(), v.data_ptr(), *layout, table.data_ptr(),
        max(table.stride(0), cols), cols, lens.data_ptr(), cu.data_ptr(), seqs, mask.data_ptr(), words, max_len,
        max_tree, dim ** -0.5 if scale is None else scale, out.data_ptr(), lse.data_ptr(), ws, ws_bytes, _stream()), "tree_attention")
    return out, lse


def _in_4_bits(k):
    """Whether k is what empty4 makes, and not bytes of another cache: uint8 [.., pages, kv_heads,
    bytes] with whole tiles of 16 rows, 272 bytes for each 32 elements of a head. No head of bytes
    up to 256 is as long; a wider one is told apart by its five dims."""
    return k.dtype is torch.uint8 and k.dim() in (3, 4) and k.size(-1) > 0 and k.size(-1) % 272 == 0


def _layers(k, v):
    """(layers, bytes from layer to layer, pages, from page to page, bytes a page, a row) of a cache."""
    if not k.is_cuda or (v is not None and not v.is_cuda):
        raise ValueError("expected device tensors")
    shape, step, size = k.shape, k.stride(), k.element_size()
    if _in_4_bits(k):  # pages as bytes of one row
        if step[-1] != 1 or (shape[-2] > 1 and step[-2] != shape[-1]):
            raise ValueError("a cache needs its pages contiguous")
        shape, step = (*shape[:-2], 1, *shape[-2:]), (*step[:-2], shape[-2] * shape[-1], *step[-2:])
    if v is not None and (v.dtype is not k.dtype or v.shape != k.shape or v.stride() != k.stride()):
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
    the copies a fork makes. src, dst int32 [n]; dst distinct and not in src. Rows of any
    type are copied; uint8 [layers, pages, kv_heads, n] is a cache in 4 bits where n is a
    multiple of 272, and else a layer of bytes (of heads that wide: [1, pages, page, kv_heads, dim])."""
    layers, layer_step, pages, page_step, page_bytes, _ = _layers(k, v)
    _int32("src", src, 1)
    _int32("dst", dst, 1)
    if src.size(0) != dst.size(0):
        raise ValueError("src and dst must be of one length")
    check(lib().spiral_cache_copy_pages(k.data_ptr(), None if v is None else v.data_ptr(), layers, layer_step, pages,
                                        page_step, page_bytes, src.data_ptr(), dst.data_ptr(), src.size(0), _stream()),
          "copy_pages")


def compact(k, v, table, lens, keep, kept, dim=None):
    """Moves the kept rows of every sequence together, in every layer of k and v (v
    may be None): the row at position lens[s] + keep[s, j] goes to lens[s] + j, for
    j < kept[s]. keep [seqs, most] int32, ascending in each row; table [seqs,
    columns], lens and kept [seqs] int32. dim: of a head, for a cache in 4 bits (uint8 without
    it is a cache of bytes, as for copy_pages). Returns the new lengths, lens + kept."""
    four = dim is not None and k.dtype is torch.uint8
    if four:
        page = _page4("k", k, dim)
    elif _in_4_bits(k):
        raise ValueError("a cache in 4 bits needs dim")
    layers, layer_step, pages, page_step, page_bytes, row_bytes = _layers(k, v)
    _int32("table", table, 2)
    _int32("lens", lens, 1)
    _int32("keep", keep, 2)
    _int32("kept", kept, 1)
    seqs = lens.size(0)
    if table.size(0) != seqs or keep.size(0) != seqs or kept.size(0) != seqs:
        raise ValueError("table, keep and kept need a row for each of lens")
    new_lens = torch.empty_like(lens)
    call, layout = lib().spiral_cache_compact, (page_bytes // row_bytes, row_bytes)
    if four:
        call, layout = lib().spiral_cache4_compact, (page, k.size(-2), dim)
    check(call(k.data_ptr(), None if v is None else v.data_ptr(), layers, layer_step, pages, page_step, *layout,
               table.data_ptr(), max(table.stride(0), table.size(1)), table.size(1), lens.data_ptr(), seqs,
               keep.data_ptr(), max(keep.stride(0), keep.size(1)), keep.size(1), kept.data_ptr(), new_lens.data_ptr(),
               _stream()), "compact")
    return new_lens


def _floats(name, t, size):
    if t.dtype is not _F32 or t.shape != (size,) or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 device tensor [{size}]")
    return t.data_ptr()


def _logits(name, t):
    shape, step = t.shape, t.stride()
    if not t.is_cuda or len(shape) != 2 or t.dtype not in _FLOATS:
        raise ValueError(f"{name} must be a 2-D float32, float16 or bfloat16 device tensor")
    if shape[1] > 1 and step[1] != 1 or shape[0] > 1 and step[0] < shape[1]:
        raise ValueError(f"{name}'s rows must be contiguous and not overlap")
    return t.data_ptr(), step[0] if shape[0] > 1 else shape[1]


def verify_workspace(logits, seqs, max_tree, draft=None):
    """Workspace for verify over logits of this shape, with or without a draft model's."""
    n = lib().spiral_draft_verify_workspace_bytes(logits.size(0), seqs, logits.size(1), draft is not None)
    if n == 0 and logits.size(0) > 0:
        raise ValueError("verify takes at most 32767 nodes, 65535 sequences and a vocabulary of 1 to 2^24 tokens")
    return torch.empty(max(n, 16), dtype=torch.uint8, device=logits.device)


def verify(logits, tokens, cu, accept, sample, *, max_tree, temperature=None, parents=None, draft=None, out=None,
           workspace=None):
    """Drafted tokens that the target's probabilities accept: (keep, kept, tokens).

    logits [nodes, vocab]: the target's behind each node of the trees that tree_attention
    took (float32, float16 or bfloat16). tokens [nodes] int32: the nodes' tokens, the first of a
    tree (at cu[s]) the last one known. parents [nodes] int32: a node's parent as an index
    in its tree (None: the node in front). draft [nodes, vocab]: the logits that a chain's
    tokens were drawn from, row i behind node i (no parents then). accept [nodes] and sample
    [seqs] float32: random numbers in [0, 1), for a node and for the token drawn at the
    end. temperature [seqs] float32 (None: 1; 0: the largest logit).

    Given tokens are accepted with their probability among what their siblings in front
    left, drawn ones with min(1, p / q); the last token comes from what is left of p. keep
    [seqs, max_tree] int32 holds the path's nodes, as compact takes them, kept [seqs] how
    many, tokens [seqs, max_tree] the accepted tokens and the drawn one, kept[s] of them, -1
    behind (and where the target's row at the path's end holds a NaN or +infinity, or no number).
    out: the three, to write to, none over another. max_tree: at least the largest tree, at
    most 1024; nodes are at most 32767, the vocabulary 2^24. workspace: verify_workspace's
    (None: its own)."""
    at, step = _logits("logits", logits)
    nodes, vocab = logits.shape
    d_at, d_step = None, 0
    if draft is not None:
        d_at, d_step = _logits("draft", draft)
        if draft.dtype is not logits.dtype or draft.shape != logits.shape:
            raise ValueError("draft must have logits' type and shape")
        if parents is not None:
            raise ValueError("a draft model's tokens are chains: parents must be None")
    for name, t in (("tokens", tokens), ("parents", parents), ("cu", cu)):
        if t is not None:
            _int32(name, t, 1)
    seqs = len(sample)
    if len(tokens) != nodes or (parents is not None and len(parents) != nodes) or len(cu) != seqs + 1:
        raise ValueError("tokens and parents need an entry for each node, cu one more than sample")
    if out is None:
        keep, said = tokens.new_empty((2, seqs, max_tree)).unbind()
        kept, keep_step = tokens.new_empty(seqs), max_tree
    else:
        keep, kept, said = out
        for name, t in (("keep", keep), ("tokens to write", said)):
            _int32(name, t, 2)
            if t.shape != (seqs, max_tree) or t.stride() != keep.stride():
                raise ValueError("keep and the tokens to write must be [seqs, max_tree], of one layout")
        _int32("kept", kept, 1)
        if len(kept) != seqs:
            raise ValueError("kept needs an entry for each of sample")
        keep_step = max(keep.stride(0), max_tree)
    if max_tree == 0:  # empty trees
        return keep, kept.zero_(), said
    if workspace is None:
        workspace = verify_workspace(logits, seqs, max_tree, draft)
    elif not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be on the device and contiguous")
    u, r = _floats("accept", accept, nodes), _floats("sample", sample, seqs)
    heat = None if temperature is None else _floats("temperature", temperature, seqs)
    check(lib().spiral_draft_verify(
        _FLOATS[logits.dtype], at, step, d_at, d_step, nodes, vocab, tokens.data_ptr(),
        None if parents is None else parents.data_ptr(), cu.data_ptr(), seqs, max_tree, u, r, heat,
        keep.data_ptr(), kept.data_ptr(), said.data_ptr(), keep_step, workspace.data_ptr(),
        workspace.nbytes, _stream()), "verify")
    return keep, kept, said


def _mass(name, t, seqs):
    shape, step = t.shape, t.stride()
    if t.dtype is not _F32 or len(shape) != 2 or not t.is_cuda or shape[0] != seqs:
        raise ValueError(f"{name} must be a float32 device tensor with a row for each sequence")
    if shape[1] > 1 and step[1] != 1 or seqs > 1 and step[0] < shape[1]:
        raise ValueError(f"{name}'s rows must be contiguous and not overlap")
    return t.data_ptr(), step[0] if seqs > 1 else shape[1], shape[1]


def row_weights(q, k, table, lens, cu, mask, lse, mass, *, max_len, max_tree, scale=None, counted=None):
    """Adds to mass [seqs, columns] (float32) the attention weight that each position of a
    sequence's cache gets from its tree's nodes, summed over nodes and heads; returns mass.

    q, k, table, lens, cu, mask, max_len, max_tree and scale as tree_attention took them, lse
    [nodes, heads] as it gave it. counted [nodes] float32: a factor for each node (None: 1; 0
    leaves it out, as for drafts that were turned down). Positions past mass are left out."""
    if not (q.is_cuda and k.is_cuda and mask.is_cuda and lse.is_cuda):
        raise ValueError("expected device tensors")
    dtype, shape, sq, sk = q.dtype, q.shape, q.stride(), k.stride()
    kind = _TYPES.get(dtype)
    four = k.dtype is torch.uint8
    if kind is None or (k.dtype is not dtype and not four):
        raise ValueError("q and k must be bfloat16 or float16, the same, or k uint8 (in 4 bits)")
    nodes, heads, dim = shape
    if dim > 1 and sq[2] != 1:
        raise ValueError("q must have a contiguous dim")
    if four:
        page = _page4("k", k, dim)
        if k.dim() != 3:
            raise ValueError("row_weights takes one layer of a cache")
        layout = (k.size(0), page, k.size(1), dim, _page_step4(k))
    else:
        pages, page, kv_heads, kdim = k.shape
        if kdim != dim or (dim > 1 and sk[3] != 1):
            raise ValueError("q and k must have one dim, contiguous")
        layout = (pages, page, kv_heads, dim, sk[0], sk[1], sk[2])
    rows = _rows4(table, lens, cu)
    mask_nodes, words = mask.shape
    if mask.dtype is not torch.int64 or mask_nodes != nodes or not mask.is_contiguous():
        raise ValueError("mask must be a contiguous int64 tensor [nodes, words]")
    if max_tree > 64 * words:
        raise ValueError("mask has too few words for max_tree")
    if lse.shape != (nodes, heads) or lse.dtype is not torch.float32 or not lse.is_contiguous():
        raise ValueError("lse must be contiguous float32 [nodes, heads]")
    factors = None if counted is None else _floats("counted", counted, nodes)
    gathered = _mass("mass", mass, lens.size(0))
    call = lib().spiral_cache4_row_weights if four else lib().spiral_cache_row_weights
    check(call(kind, q.data_ptr(), sq[0], sq[1], nodes, heads, k.data_ptr(), *layout, *rows, mask.data_ptr(), words,
               max_len, max_tree, dim ** -0.5 if scale is None else scale, lse.data_ptr(), factors, *gathered,
               _stream()), "row_weights")
    return mass


def evict_workspace(mass):
    """Workspace for evict over mass of this shape, or None where it uses none."""
    n = lib().spiral_cache_evict_workspace_bytes(mass.size(1), mass.size(0))
    return torch.empty(n, dtype=_U8, device=mass.device) if n > 0 else None


def evict(mass, lens, budget, *, sinks=0, recent=0, workspace=None):
    """The rows of each sequence that stay where it has more than `budget`: the first `sinks`,
    the last `recent`, and of the others those of the largest mass (of equal ones the
    first): (keep, kept, new_mass).

    mass [seqs, columns] float32, lens [seqs] int32. keep [seqs, budget] int32: their
    positions, ascending, -1 behind; kept [seqs] how many: compact(k, v, table, zeros, keep,
    kept) moves the rows together. new_mass: mass of the rows that stay, in their new places,
    zeros behind. workspace: evict_workspace's (None: its own)."""
    _int32("lens", lens, 1)
    if budget < 0:
        raise ValueError("budget must not be negative")
    seqs = len(lens)
    at, step, cols = _mass("mass", mass, seqs)
    keep, kept, new = lens.new_empty((seqs, budget)), lens.new_empty(seqs), mass.new_empty((seqs, cols))
    if workspace is None:
        workspace = evict_workspace(mass) if cols > 16384 else None  # shorter ones are never divided
    elif not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be on the device and contiguous")
    ws, ws_bytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.nbytes)
    check(lib().spiral_cache_evict(at, step, cols, lens.data_ptr(), seqs, budget, sinks, recent, keep.data_ptr(), budget,
                                   kept.data_ptr(), new.data_ptr(), cols, ws, ws_bytes, _stream()), "evict")
    return keep, kept, new


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

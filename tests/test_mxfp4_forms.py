"""MXFP4 weights through the forms that large batches and experts take: the product that
dequantizes the weights once, the streaming passes of MUL_MAT_ID, its fused GLU in both
layouts and the ggml nodes, and blocks whose scale byte is special in all of them.

Tolerances are those of a sum of exact products (check_product); a fused GLU is held to
the unfused calls bit for bit.
"""

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_MXFP4, ggml, lib, ops, row_bytes
from test_mxfp4 import blocks, check_product, planar, rows_of, values

pytestmark = pytest.mark.gpu


def takes_dense(m, n, k):
    return lib().spiral_mul_mat_workspace_bytes(TYPE_MXFP4, n, k, m) == n * k * 2


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k,dense", [(257, 7001, 256, True), (513, 2500, 512, False), (1025, 7001, 256, True),
                                         (1300, 4501, 1152, True), (2049, 2500, 512, True), (2049, 7001, 1024, True)])
def test_dequantize_once(cuda, m, n, k, dense, out_dtype):
    """Shapes on both sides of the line; ragged rows of x and W, wider rows of both."""
    assert takes_dense(m, n, k) == dense
    raw = blocks(n, k, m + n)
    x = rows_of(m, k + 8, k, cuda)[:, :k]
    out = torch.full((m, n + 3), 7.0, dtype=out_dtype, device=cuda)
    ops.mul_mat(TYPE_MXFP4, planar(raw, cuda), n, k, x, out=out[:, :n])
    check_product(out[:, :n], x.double().cpu().numpy(), values(raw).reshape(n, k))
    assert (out[:, n:] == 7).all()


def test_dequantize_once_in_chunks(cuda):
    """A matrix past the workspace's 256 MiB of bf16: rows on both sides of the chunks' border."""
    m, n, k = 1500, 8500, 16384
    assert lib().spiral_mul_mat_workspace_bytes(TYPE_MXFP4, n, k, m) == 4352 * k * 2
    raw = blocks(n, k, 3)
    x = rows_of(m, k, 4, cuda)
    y = ops.mul_mat(TYPE_MXFP4, planar(raw, cuda), n, k, x, out_dtype=torch.float32)
    rows = np.r_[0:4, 4348:4356, 8496:8500]
    check_product(y[:, torch.from_numpy(rows).to(cuda)], x.double().cpu().numpy(), values(raw[rows]).reshape(-1, k))


@pytest.mark.parametrize("m,n,k", [(1, 20, 96), (7, 40, 4128), (16, 130, 544), (40, 300, 544), (130, 70, 1056),
                                   (300, 260, 4096), (2049, 2500, 512)])
def test_special_scales_times_bf16_rows(cuda, m, n, k):
    """Scale bytes 255 in a row's first and last block (in front of the next row's, and of
    what lies past the end of a ragged step), 0 and 254: NaN in the marked rows alone,
    the others as they are."""
    raw = blocks(n, k, 5)
    bad = [n // 2, n - 1]
    raw[bad[0], -1, 0] = raw[bad[1], 0, 0] = 255
    raw[1, 0, 0], raw[2, 0, 0] = 0, 254
    raw[2, 0, 1:] &= 0x33  # at most 1.5 * 2^127: values that bf16 holds
    raw[2, 0, 1:] |= 0x11  # and none of them zero
    x = rows_of(m, k, 6, cuda) * 2.0 ** -10
    y = ops.mul_mat(TYPE_MXFP4, planar(raw, cuda), n, k, x, out_dtype=torch.float32)
    fine = np.setdiff1d(np.arange(n), bad)
    assert torch.isnan(y[:, bad]).all()
    check_product(y[:, torch.from_numpy(fine).to(cuda)], x.double().cpu().numpy(), values(raw[fine]).reshape(-1, k))


# ---- experts ------------------------------------------------------------------------


def experts(n_expert, n, k, seed, dev):
    """(canonical blocks, planar matrices, bytes from one to the next)."""
    raw = np.stack([blocks(n, k, seed + e) for e in range(n_expert)])
    per = -(-row_bytes(TYPE_MXFP4, k) * n // 16) * 16
    return raw, planar_stack(raw, per, dev), per


def planar_stack(raw, per, dev):
    w = torch.zeros((len(raw), per), dtype=torch.uint8, device=dev)
    for e, r in enumerate(raw):
        p = planar(r, dev)
        w[e, :p.numel()] = p
    return w


def routes(n_expert, tokens, top_k, seed):
    rng = np.random.default_rng(seed)
    return np.stack([rng.choice(n_expert, top_k, replace=False) for _ in range(tokens)]).astype(np.int32)


def check_experts(got, x, raw, ids):
    xs, (n, k) = x.double().cpu().numpy(), (raw.shape[1], 32 * raw.shape[2])
    assert not got.float().cpu().numpy()[(ids < 0) | (ids >= len(raw))].any()
    for e in range(len(raw)):
        t, s = np.nonzero(ids == e)
        if t.size:
            check_product(got[t, s], xs[t, s % xs.shape[1]], values(raw[e]).reshape(n, k))


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n_expert,tokens,top_k,n,k,slots", [
    (8, 160, 2, 104, 768, 1),   # passes of 64 tokens
    (8, 100, 2, 64, 2048, 1),   # of 32
    (4, 200, 1, 32, 4096, 1),   # of 16, over pass lanes
    (16, 700, 2, 48, 544, 2),   # routed by the counting sort; a row for each slot; a ragged step
    (32, 1100, 8, 64, 256, 1),  # lists past LDS
    (6, 3, 4, 40, 2880, 1),     # decoding
])
def test_experts(cuda, n_expert, tokens, top_k, n, k, slots, out_dtype):
    raw, w, per = experts(n_expert, n, k, 40, cuda)
    ids = routes(n_expert, tokens, top_k, tokens)
    ids[::13, 0], ids[1::17, -1] = -1, n_expert + 3
    if tokens > 600:
        ids[:500, 0] = 3
    x = rows_of(tokens * slots, k, 7, cuda).view(tokens, slots, k)
    got = ops.mul_mat_id(TYPE_MXFP4, w, per, n_expert, n, k, x, torch.from_numpy(ids).to(cuda), out_dtype=out_dtype)
    check_experts(got, x, raw, ids)


@pytest.mark.parametrize("n_expert,tokens,top_k,F,k", [(8, 1, 3, 72, 96), (8, 40, 3, 72, 544), (6, 30, 2, 40, 2880),
                                                       (12, 160, 8, 40, 256), (8, 300, 2, 48, 512)])
@pytest.mark.parametrize("split", [False, True])
def test_fused_glu_equals_the_unfused_calls(cuda, n_expert, tokens, top_k, F, k, split):
    ids = routes(n_expert, tokens, top_k, tokens)
    ids[::7, 0], ids[3::11, -1] = -1, 99
    idd, x = torch.from_numpy(ids).to(cuda), rows_of(tokens, k, 8, cuda).view(tokens, 1, k)
    (raw_g, wg, per), (raw_u, wu, _) = experts(n_expert, F, k, 60, cuda), experts(n_expert, F, k, 90, cuda)
    pg, pu = (ops.mul_mat_id(TYPE_MXFP4, w, per, n_expert, F, k, x, idd, out_dtype=torch.float32) for w in (wg, wu))
    check_experts(pg, x, raw_g, ids)
    both = np.concatenate([raw_g, raw_u], axis=1)
    per2 = -(-row_bytes(TYPE_MXFP4, k) * 2 * F // 16) * 16
    merged = planar_stack(both, per2, cuda)
    for op in (ops.GLU_REGLU, ops.GLU_GEGLU, ops.GLU_SWIGLU, ops.GLU_GEGLU_ERF, ops.GLU_GEGLU_QUICK):
        for swapped in (False, True):
            want = ops.glu_split(pg, pu, op, swapped)
            for dtype in (torch.float32, torch.bfloat16):
                if split:
                    got = ops.mul_mat_id_glu_split(TYPE_MXFP4, wg, wu, per, n_expert, F, k, x, idd, op, swapped, dtype)
                else:
                    got = ops.mul_mat_id_glu(TYPE_MXFP4, merged, per2, n_expert, 2 * F, k, x, idd, op, swapped, dtype)
                assert torch.equal(got, want.to(dtype)), (op, swapped, dtype)


@pytest.mark.parametrize("tokens,k", [(2, 96), (40, 544), (700, 160)])
def test_special_scales_of_experts(cuda, tokens, k):
    """NaN blocks at the end of a row, ragged steps behind it: that row's results alone."""
    n_expert, n = 4, 40
    raw, w, per = experts(n_expert, n, k, 70, cuda)
    raw[:, 11, -1, 0], raw[:, 39, -1, 0], raw[:, 3, 0, 0] = 255, 255, 0
    w = planar_stack(raw, per, cuda)
    ids = routes(n_expert, tokens, 2, 5)
    x = rows_of(tokens, k, 9, cuda).view(tokens, 1, k)
    got = ops.mul_mat_id(TYPE_MXFP4, w, per, n_expert, n, k, x, torch.from_numpy(ids).to(cuda), out_dtype=torch.float32)
    fine = np.setdiff1d(np.arange(n), [11, 39])
    assert torch.isnan(got[..., [11, 39]]).all()
    check_experts(got[..., torch.from_numpy(fine).to(cuda)], x, raw[:, fine], ids)


# ---- ggml ---------------------------------------------------------------------------


def test_ggml_experts(cuda):
    """MUL_MAT_ID nodes over MXFP4 experts, and the split GLU that graph_compute fuses (up,
    gate, GLU: neither product is written); flagged OUTPUT a product is, with the same bits."""
    k, F, n_expert, top_k, tokens = 160, 48, 5, 2, 9
    raws = [np.stack([blocks(F, k, s + e) for e in range(n_expert)]) for s in (10, 30)]
    ids = routes(n_expert, tokens, top_k, 1)
    x = rows_of(tokens, k, 2, "cpu").float()
    buf = ggml.Buffer(4 << 20)
    ag, au = (buf.alloc(ggml.new_tensor(TYPE_MXFP4, [k, F, n_expert])) for _ in raws)
    for t, r in zip((ag, au), raws):
        buf.set(t, r.tobytes())
        assert bytes(buf.get(t)) == r.tobytes()
    b = buf.alloc(ggml.new_tensor(ggml.TYPE_F32, [k, 1, tokens]))
    buf.set(b, x.numpy().tobytes())
    it = buf.alloc(ggml.new_tensor(ggml.TYPE_I32, [top_k, tokens]))
    buf.set(it, ids.tobytes())
    up, gate = (buf.alloc(ggml.mul_mat_id(w, b, it, name=n)) for w, n in ((au, "ffn_up"), (ag, "ffn_gate")))
    g = buf.alloc(ggml.glu_split(gate, up, ggml.GLU_SWIGLU))
    assert all(ggml.supports_op(t) for t in (up, gate, g))
    sentinel = np.full(F * top_k * tokens, 7.0, dtype=np.float32).tobytes()
    for t in (up, gate):
        buf.set(t, sentinel)
    be = ggml.Backend(0)
    assert be.graph_compute([up, gate, g]) == 0
    be.synchronize()
    assert buf.get(up) == sentinel and buf.get(gate) == sentinel
    fused = bytes(buf.get(g))
    gate.flags = up.flags = ggml.FLAG_OUTPUT
    assert be.graph_compute([up, gate, g]) == 0
    be.synchronize()
    assert bytes(buf.get(g)) == fused
    for t, r in zip((gate, up), raws):
        got = torch.from_numpy(np.frombuffer(buf.get(t), dtype=np.float32).reshape(tokens, top_k, F).copy())
        check_experts(got, x.view(tokens, 1, k), r, ids)
    be.free()
    buf.free()

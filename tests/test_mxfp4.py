"""MXFP4 (SPIRAL_TYPE_MXFP4): the format against a numpy restatement of the OCP
rule, its products against float64.

Tolerance of a product. Every term x W is exact in fp32 (x bf16 or E2M1, W
E2M1 times a power of two), so an F32 result is off by its sum alone: whatever
the order of its k terms, by at most k half steps (2^-24) of the sum of their
magnitudes. A bf16 result adds its own rounding, 2^-8 of the value at most.
"""

import ctypes

import numpy as np
import pytest
import torch

from spiral_amd import TYPE_BF16, TYPE_F32, TYPE_MXFP4, _lib, ggml, lib, ops, row_bytes

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


# ---- the format, restated -----------------------------------------------------


def values(raw):
    """Canonical blocks [..., 17] -> float64 [..., 32]."""
    e = raw[..., :1].astype(np.float64) - 127
    q = raw[..., 1:]
    v = E2M1[np.concatenate([q & 15, q >> 4], axis=-1)] * np.exp2(e)
    return np.where(raw[..., :1] == 255, np.nan, v)


def quantize(x):
    """float64 rows [rows, k] -> canonical blocks [rows, k / 32, 17]."""
    b = x.reshape(x.shape[0], -1, 32)
    top = np.abs(b).max(axis=-1)
    with np.errstate(all="ignore"):
        e = np.where(top > 0, np.frexp(top)[1] - 3, -127).clip(-127, 127)
        a = np.abs(b) / np.exp2(e.astype(np.float64))[..., None]
        code = np.zeros(b.shape, dtype=np.uint8)
        for c in range(7):  # a tie between c and c + 1 goes to the even of them
            border = (E2M1[c] + E2M1[c + 1]) / 2
            code += (a >= border) if c % 2 else (a > border)
    code |= np.where(np.signbit(b), 8, 0).astype(np.uint8)
    raw = np.empty(b.shape[:2] + (17,), dtype=np.uint8)
    raw[..., 0] = (e + 127).astype(np.uint8)
    raw[..., 1:] = code[..., :16] | (code[..., 16:] << 4)
    raw[~np.isfinite(top)] = 0
    raw[~np.isfinite(top), 0] = 255
    return raw


def blocks(n, k, seed, lo=118, hi=130):
    rng = np.random.default_rng(seed)
    raw = rng.integers(0, 256, (n, k // 32, 17), dtype=np.uint8)
    raw[..., 0] = rng.integers(lo, hi, (n, k // 32))
    return raw


def planar(raw, dev):
    n, nb, _ = raw.shape
    return ops.to_planar(TYPE_MXFP4, torch.from_numpy(raw.reshape(-1).copy()).to(dev), n, 32 * nb)


def canonical(p, n, k):
    return ops.from_planar(TYPE_MXFP4, p, n, k).cpu().numpy().reshape(n, k // 32, 17)


def rows_of(m, k, seed, dev, dtype=torch.bfloat16):
    gen = torch.Generator().manual_seed(seed)
    return torch.randn((m, k), generator=gen).to(dtype).to(dev)


def check_product(got, x, w):
    """got against float64 rows x [m, k] and w [n, k]."""
    y, mag = x @ w.T, np.abs(x) @ np.abs(w).T
    tol = x.shape[1] * 2.0 ** -24 * mag
    if got.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * np.abs(y)
    err = np.abs(got.double().cpu().numpy() - y)
    assert (err <= tol).all(), (err - tol).max()


# ---- refusals (no device needed) ------------------------------------------------


def test_sizes(spiral_lib):
    L = spiral_lib
    assert L.spiral_row_bytes(TYPE_MXFP4, 4096) == 2176 and row_bytes(TYPE_MXFP4, 32) == 17
    assert L.spiral_row_bytes(TYPE_MXFP4, 48) == 0
    assert L.spiral_tensor_bytes(TYPE_MXFP4, 3, 96) == 153
    for m in (1, 2, 16):
        assert L.spiral_mul_mat_workspace_bytes(TYPE_MXFP4, 4096, 4096, m) == 0
    assert L.spiral_mul_mat_workspace_bytes(TYPE_MXFP4, 4096, 4096, 17) == 32 * 4096 * 2
    assert L.spiral_gemv_relaxed_max_k(TYPE_MXFP4) == 0


def test_refusals(spiral_lib):
    L = spiral_lib
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    bf, f32 = TYPE_BF16, TYPE_F32
    assert L.spiral_mxfp4_quantize(p, TYPE_MXFP4, 64, 2, 64, p, None) == 6
    assert L.spiral_mxfp4_quantize(p, bf, 48, 2, 48, p, None) == 1        # k not a multiple of 32
    assert L.spiral_mxfp4_quantize(p, bf, 32, 2, 64, p, None) == 1        # stride below k
    assert L.spiral_mxfp4_quantize(p, bf, 64, -1, 64, p, None) == 1
    assert L.spiral_mxfp4_quantize(p, bf, 64, 1 << 62, 64, p, None) == 1
    assert L.spiral_mxfp4_quantize(None, bf, 64, 2, 64, p, None) == 3
    assert L.spiral_mxfp4_quantize(p, bf, 64, 2, 64, None, None) == 3
    assert L.spiral_mxfp4_quantize(odd, bf, 64, 2, 64, p, None) == 2
    assert L.spiral_mxfp4_quantize(p, bf, 68, 2, 64, p, None) == 2
    assert L.spiral_mxfp4_quantize(None, bf, 64, 0, 64, None, None) == 0  # no rows: a no-op
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, p, TYPE_MXFP4, 4, None, 0, None) == 6
    assert L.spiral_mxfp4_mul_mat(None, 4, 64, p, 2, p, bf, 4, None, 0, None) == 3
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, None, bf, 4, None, 0, None) == 3
    assert L.spiral_mxfp4_mul_mat(p, 4, 60, p, 2, p, bf, 4, None, 0, None) == 1
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 0, p, bf, 4, None, 0, None) == 1
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, p, bf, 3, None, 0, None) == 1  # ldy below n_rows
    assert L.spiral_mxfp4_mul_mat(p, 1 << 61, 64, p, 2, p, bf, 1 << 61, None, 0, None) == 1
    assert L.spiral_mxfp4_mul_mat(odd, 4, 64, p, 2, p, bf, 4, None, 0, None) == 2
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, p, bf, 4, odd, 64, None) == 2
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, p, bf, 4, p, -1, None) == 1
    assert L.spiral_mxfp4_mul_mat_workspace_bytes(4, 60, 100) == 0 and L.spiral_mxfp4_mul_mat_workspace_bytes(4096, 4096, 16) == 0
    assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, ctypes.c_void_p(4098), f32, 4, None, 0, None) == 2
    assert L.spiral_gemv_relaxed(TYPE_MXFP4, p, 4, 64, p, p, bf, None) == 1
    assert L.spiral_to_planar(TYPE_MXFP4, p, 33, 2, 64, p, None) == 1     # stride below the row
    if L.spiral_device_count() == 0:
        assert L.spiral_mxfp4_quantize(p, bf, 64, 2, 64, p, None) == 4
        assert L.spiral_mxfp4_mul_mat(p, 4, 64, p, 2, p, bf, 4, None, 0, None) == 4
        assert L.spiral_to_planar(TYPE_MXFP4, p, 35, 2, 64, p, None) == 4  # an odd stride is a stride
        assert L.spiral_mul_mat(TYPE_MXFP4, p, 4, 64, p, 64, 1, p, f32, 4, None, 0, None) == 4


def test_wrapper_refusals():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device tensor"):
        ops.mxfp4_quantize(x)


# ---- the format on the GPU --------------------------------------------------------


@pytest.mark.gpu
def test_every_scale_and_code(cuda):
    raw = np.empty((256, 1, 17), dtype=np.uint8)
    raw[:, 0, 0] = np.arange(256)
    raw[:, 0, 1:] = np.arange(16) | ((15 - np.arange(16)) << 4)
    with np.errstate(over="ignore"):
        want = values(raw).reshape(256, 32).astype(np.float32)  # past the range: infinity
    w = planar(raw, cuda)
    got = ops.dequant(TYPE_MXFP4, w, 256, 32).float().cpu().numpy()
    assert np.array_equal(got.view(np.uint32)[:255], want.view(np.uint32)[:255])  # signs of zeros too
    assert np.isnan(got[255]).all()
    ids = torch.tensor([5, -1, 200, 256], device=cuda)
    rows = ops.get_rows(TYPE_MXFP4, w, 256, 32, ids).cpu().numpy()
    assert np.array_equal(rows[[0, 2]], want[[5, 200]]) and not rows[[1, 3]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 1, 6])
def test_layout_round_trip(cuda, pad):
    """Rows at odd byte strides, from an odd address."""
    n, k = 5, 96
    raw = blocks(n, k, 1)
    stride = row_bytes(TYPE_MXFP4, k) + pad
    src = torch.zeros(n * stride + 1, dtype=torch.uint8, device=cuda)[1:]
    src.view(n, stride)[:, :51] = torch.from_numpy(raw.reshape(n, 51)).to(cuda)
    p = ops.to_planar(TYPE_MXFP4, src, n, k, row_stride=stride)
    flat = p.cpu().numpy()
    assert np.array_equal(flat[:16 * 15].reshape(15, 16), raw.reshape(15, 17)[:, 1:])
    assert np.array_equal(flat[16 * 15:], raw.reshape(15, 17)[:, 0])
    back = ops.from_planar(TYPE_MXFP4, p, n, k, row_stride=stride)
    assert torch.equal(back.view(n, stride)[:, :51], src.view(n, stride)[:, :51])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k,pad", [(1, 32, 0), (1, 4096, 8), (3, 96, 0), (7, 2080, 24), (130, 256, 0)])
def test_quantize(cuda, dtype, m, k, pad):
    buf = rows_of(m, k + pad, 3 * m + k, cuda, dtype) * 3
    x = buf[:, :k]
    got = canonical(ops.mxfp4_quantize(x), m, k)
    assert np.array_equal(got, quantize(x.double().cpu().numpy()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_edges(cuda, dtype):
    """Ties and saturation under scales over the whole range, zeros, subnormals,
    the largest numbers, infinities and NaN."""
    grid = np.concatenate([np.arange(0, 8, 0.25), [5, 7, 0.125, 7.9375]])
    rows = []
    for e in (-133, -127, -126, -100, -3, 0, 9, 100, 124):
        for top in (4, 6, 7.5):
            r = np.resize(grid, 32) * np.where(np.arange(32) % 3 == 1, -1, 1)
            r = np.minimum(np.abs(r), top) * np.sign(r)
            r[0] = top
            rows.append(r * 2.0 ** e)
    rows.append(np.zeros(32))
    rows.append(np.where(np.arange(32) == 7, -0.0, 0.0))
    fin = torch.finfo(dtype)
    rows.append(np.where(np.arange(32) == 3, fin.max, fin.max / 2))
    rows.append(np.where(np.arange(32) == 30, fin.tiny / 8, 0))
    for bad in (np.inf, -np.inf, np.nan):
        for at in (0, 5, 17, 31):
            rows.append(np.where(np.arange(32) == at, bad, 1.0))
    x = torch.from_numpy(np.stack(rows)).to(dtype).to(cuda)
    assert np.array_equal(canonical(ops.mxfp4_quantize(x), len(rows), 32), quantize(x.double().cpu().numpy()))


@pytest.mark.gpu
def test_quantize_into_a_buffer_and_no_rows(cuda):
    x = rows_of(3, 64, 5, cuda)
    buf = torch.full((200,), 77, dtype=torch.uint8, device=cuda)
    assert ops.mxfp4_quantize(x, out=buf) is buf
    assert np.array_equal(canonical(buf[:102], 3, 64), quantize(x.double().cpu().numpy()))
    assert (buf[102:] == 77).all()
    assert ops.mxfp4_quantize(x[:0]).numel() == 0
    with pytest.raises(ValueError, match="at least"):
        ops.mxfp4_quantize(x, out=buf[:101])
    with pytest.raises(ValueError, match="2-D"):
        ops.mxfp4_quantize(x.t())


# ---- products -----------------------------------------------------------------------

SHAPES = [(1, 1, 32), (1, 37, 4096), (2, 16, 96), (5, 100, 160), (16, 33, 1056), (16, 130, 14336), (17, 40, 128),
          (33, 257, 544), (65, 100, 2080), (130, 70, 512)]


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES + [(3, 12300, 96), (16, 12345, 1056), (300, 260, 4096), (513, 512, 1024)])
def test_mul_mat_bf16_rows(cuda, m, n, k, out_dtype):
    raw = blocks(n, k, m + n)
    x = rows_of(m, k + 8, k, cuda)[:, :k]  # rows of a wider tensor
    out = torch.full((m, n + 3), 7.0, dtype=out_dtype, device=cuda)
    ops.mul_mat(TYPE_MXFP4, planar(raw, cuda), n, k, x, out=out[:, :n])
    check_product(out[:, :n], x.double().cpu().numpy(), values(raw).reshape(n, k))
    assert (out[:, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES + [(1, 12290, 288), (9, 12345, 1056), (64, 64, 256), (257, 300, 1536), (300, 520, 4096), (1000, 129, 288)])
def test_mul_mat_mxfp4_rows(cuda, m, n, k, out_dtype):
    raw, xr = blocks(n, k, m + n), blocks(m, k, 7 * m + k)
    out = torch.full((m, n + 5), 7.0, dtype=out_dtype, device=cuda)
    ops.mxfp4_mul_mat(planar(raw, cuda), n, k, planar(xr, cuda), m, out=out[:, :n])
    check_product(out[:, :n], values(xr).reshape(m, k), values(raw).reshape(n, k))
    assert (out[:, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(50, 131, 14336), (200, 300, 5152), (17, 64, 8224)])
def test_mul_mat_over_ranges_of_k(cuda, m, n, k, out_dtype):
    """Too few tiles for the GPU: ranges of k joined from the workspace, from less
    of it and without it, into rows of any alignment."""
    raw, xr = blocks(n, k, m + n), blocks(m, k, 7 * m + k)
    w, x = planar(raw, cuda), planar(xr, cuda)
    ws = ops.mxfp4_mul_mat_workspace(n, k, m, cuda)
    ws.fill_(0xFF)
    for part in (ws, ws[:ws.numel() // 2], ws[:16]):
        out = torch.full((m, n + 3), 7.0, dtype=out_dtype, device=cuda)
        ops.mxfp4_mul_mat(w, n, k, x, m, out=out[:, :n], workspace=part)
        check_product(out[:, :n], values(xr).reshape(m, k), values(raw).reshape(n, k))
        assert (out[:, n:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 20, 96), (16, 40, 4096), (80, 90, 544), (300, 300, 1024), (40, 90, 5152)])
def test_nan_blocks_stay_in_their_rows(cuda, m, n, k):
    """A NaN block, the last block of its row (in front of the next row's scales
    and of what lies past the end of a ragged step): its row or column is NaN,
    everything else is what it was."""
    raw, xr = blocks(n, k, 2), blocks(m, k, 3)
    for r in (raw, xr):
        r[r.shape[0] // 2, -1, 0] = 255
        r[r.shape[0] // 2, 0, 0] = 255
    got = ops.mxfp4_mul_mat(planar(raw, cuda), n, k, planar(xr, cuda), m, out_dtype=torch.float32).cpu().numpy()
    w, x = values(raw).reshape(n, k), values(xr).reshape(m, k)
    assert np.array_equal(np.isnan(got), np.isnan(x @ w.T))
    ok = ~np.isnan(got)
    mag = np.abs(x) @ np.abs(w).T
    assert (np.abs(got - x @ w.T)[ok] <= (k * 2.0 ** -24 * mag)[ok]).all()
    xb = rows_of(m, k, 4, cuda)
    xb[m // 2, k - 1] = float("nan")
    xb[0, 0] = float("inf") if m > 1 else 1.0
    wf = blocks(n, k, 5)
    wf[..., 1:] &= 0x77  # no negative codes: infinity times a weight is infinity or, at code 0, NaN
    got = ops.mul_mat(TYPE_MXFP4, planar(wf, cuda), n, k, xb, out_dtype=torch.float32).cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = xb.double().cpu().numpy() @ values(wf).reshape(n, k).T
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.isinf(got), np.isinf(want))


@pytest.mark.gpu
def test_scales_at_the_ends_of_their_range(cuda):
    """Scale bytes 0 and 254 against each other, and products below float32's
    range, which vanish."""
    n, k, m = 20, 160, 18
    raw, xr = blocks(n, k, 1, 0, 1), blocks(m, k, 2, 254, 255)
    got = ops.mxfp4_mul_mat(planar(raw, cuda), n, k, planar(xr, cuda), m, out_dtype=torch.float32)
    check_product(got, values(xr).reshape(m, k), values(raw).reshape(n, k))
    low = planar(blocks(m, k, 3, 0, 2), cuda)
    assert not ops.mxfp4_mul_mat(planar(raw, cuda), n, k, low, m, out_dtype=torch.float32).any()


@pytest.mark.gpu
def test_row_is_independent_of_the_batch(cuda):
    """Every form multiplies the same exact weights: F32 results of one row differ
    by the order of their sums alone."""
    n, k = 96, 1024
    raw = blocks(n, k, 9)
    w, x = planar(raw, cuda), rows_of(300, k, 10, cuda)
    tol = 2 * k * 2.0 ** -24 * (np.abs(x[:1].double().cpu().numpy()) @ np.abs(values(raw).reshape(n, k)).T)
    one = ops.mul_mat(TYPE_MXFP4, w, n, k, x[:1], out_dtype=torch.float32)
    for m in (2, 16, 17, 300):
        got = ops.mul_mat(TYPE_MXFP4, w, n, k, x[:m], out_dtype=torch.float32)
        assert (np.abs((got[:1] - one).cpu().numpy()) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,n_expert,n,k", [(1, 4, 40, 96), (10, 6, 64, 512), (300, 3, 96, 1056), (40, 3, 50, 4160)])
def test_mul_mat_id(cuda, tokens, n_expert, n, k):
    raw = np.stack([blocks(n, k, 20 + e) for e in range(n_expert)])
    per = -(-row_bytes(TYPE_MXFP4, k) * n // 16) * 16
    w = torch.zeros((n_expert, per), dtype=torch.uint8, device=cuda)
    for e in range(n_expert):
        w[e, :n * row_bytes(TYPE_MXFP4, k)] = planar(raw[e], cuda)
    x = rows_of(tokens, k, 1, cuda)
    ids = torch.randint(0, n_expert, (tokens, 2), generator=torch.Generator().manual_seed(2), dtype=torch.int32)
    ids[0, 1] = -1
    got = ops.mul_mat_id(TYPE_MXFP4, w, per, n_expert, n, k, x.view(tokens, 1, k), ids.to(cuda),
                         out_dtype=torch.float32)
    assert not got[0, 1].any()
    xs = x.double().cpu().numpy()
    for e in range(n_expert):
        t, s = np.nonzero(ids.numpy() == e)
        if t.size:
            check_product(got[t, s], xs[t], values(raw[e]).reshape(n, k))
    if k <= 4096 and n % 2 == 0:
        fused = ops.mul_mat_id_glu(TYPE_MXFP4, w, per, n_expert, n, k, x.view(tokens, 1, k), ids.to(cuda),
                                   out_dtype=torch.float32).double().cpu().numpy()
        assert not fused[0, 1].any()
        for e in range(n_expert):
            t, s = np.nonzero(ids.numpy() == e)
            v = values(raw[e]).reshape(n, k)
            y, tol = xs[t] @ v.T, k * 2.0 ** -24 * (np.abs(xs[t]) @ np.abs(v).T)
            (g, u), (tg, tu) = np.split(y, 2, axis=1), np.split(tol, 2, axis=1)
            silu = g / (1 + np.exp(-g))
            # silu's slope is below 1.1; 2^-20 of the value for its exponential, division and two products
            assert (np.abs(fused[t, s] - silu * u) <=
                    1.1 * tg * (np.abs(u) + tu) + np.abs(silu) * tu + 2.0 ** -20 * np.abs(silu * u)).all()


@pytest.mark.gpu
def test_ggml_graph(cuda):
    """MUL_MAT and GET_ROWS nodes over a canonical tensor, and partial writes."""
    n, k, m = 48, 96, 3
    raw = blocks(n, k, 31)
    buf = ggml.Buffer(1 << 16)
    w = buf.alloc(ggml.new_tensor(TYPE_MXFP4, [k, n], "w"))
    data = raw.tobytes()
    buf.set(w, data)
    assert bytes(buf.get(w)) == data
    buf.set(w, data[100:777], offset=100)  # a range of whole and cut blocks
    assert bytes(buf.get(w)) == data and bytes(buf.get(w, 50, 33)) == data[33:83]
    ids = torch.tensor([7, 0, 47], dtype=torch.int32, device=cuda)
    it = ggml.new_tensor(ggml.TYPE_I32, [m], "ids")
    it.data = ids.data_ptr()
    x = ggml.get_rows(w, it)
    y = ggml.mul_mat(w, x)
    mem = []
    for node in (x, y):
        mem.append(torch.empty((m, node.ne[0]), dtype=torch.float32, device=cuda))
        node.data = mem[-1].data_ptr()
    torch.cuda.synchronize()
    be = ggml.Backend(0)
    assert be.graph_compute([x, y]) == 0
    be.synchronize()
    v = values(raw).reshape(n, k)
    assert np.array_equal(mem[0].cpu().numpy(), v[[7, 0, 47]])
    check_product(mem[1], v[[7, 0, 47]], v)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 70, 300])
def test_captured_and_on_another_stream(cuda, m):
    """Quantization and both products recorded in a HIP graph on a side stream,
    replayed on new inputs with eager calls in between."""
    n, k = 300, 512
    w = planar(blocks(n, k, 1), cuda)
    x = rows_of(m, k, 2, cuda)
    q = torch.empty(m * row_bytes(TYPE_MXFP4, k), dtype=torch.uint8, device=cuda)
    y4, y16 = (torch.empty((m, n), dtype=torch.float32, device=cuda) for _ in range(2))
    ws = ops.mul_mat_workspace(TYPE_MXFP4, n, k, m, cuda)

    def call(a, b):
        ops.mxfp4_quantize(x, out=q)
        ops.mxfp4_mul_mat(w, n, k, q, m, out=a)
        ops.mul_mat(TYPE_MXFP4, w, n, k, x, out=b, workspace=ws)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(y4, y16)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(y4, y16)
    for seed in range(4):
        x.copy_(rows_of(m, k, 10 + seed, cuda))
        y4.fill_(float("nan"))
        y16.fill_(float("nan"))
        graph.replay()
        got4, got16 = y4.clone(), y16.clone()
        want4, want16 = torch.empty_like(y4), torch.empty_like(y16)
        call(want4, want16)
        torch.cuda.synchronize()
        assert torch.equal(got4, want4) and torch.equal(got16, want16)


def test_status_names():
    assert _lib.STATUS[1] == "SPIRAL_ERR_SHAPE" and lib().spiral_status_string(1)

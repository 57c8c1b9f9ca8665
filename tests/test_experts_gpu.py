"""The expert-layer operators (include/gpuq.h: gpuq_mxfp4_*, gpuq_route_*) against plain implementations in 64 bits:
rounding to MXFP4 code by code, products at the sizes where tiles, k pieces and groups end, routing with ties and
nothing left, grouping, streams, graphs, 32-bit limits and refusals.

Tolerances: a product's f32 sum of K exact terms is off by at most (K + 8) 2^-23 sum |x w| in any order, and rounding the
output adds half a unit of its type (2^-24, 2^-11, 2^-8 of the value, and half the smallest F16 step). Scores are a few
correctly rounded f32 operations around expf (2 units): 32 units in all. Codes, ids and orders are exact."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

F32, F16, Q8_0, BF16, MXFP4 = 0, 1, 8, 30, 39
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


@pytest.fixture(scope="module")
def gq():
    import torch
    torch.cuda.init()
    import gpuq
    return gpuq.load_gpuq(0)


@pytest.fixture(scope="module")
def ex(gq):
    from gpuq import experts
    return experts


def torch_():
    import torch
    return torch


def dtype(name):
    torch = torch_()
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


# ---------------------------------------------------------------- plain implementations
def round_blocks(x):
    """f64 [n, ncol] -> (codes [n, ncol], exponents [n, ncol / 32]): nearest by distance, the smaller on a tie"""
    n, ncol = x.shape
    b = np.where(np.isnan(x), 0.0, x).reshape(n, ncol // 32, 32)
    top = np.abs(b).max(axis=2)
    with np.errstate(divide="ignore"):
        e = np.where(np.isinf(top), 252, np.where(top > 0, np.frexp(top)[1] - 1 - 2 + 127, 0))
    e = np.clip(e, 0, 252)
    t = np.minimum(np.abs(b), 1e300) / np.exp2(e.astype(np.float64) - 127)[..., None]
    code = np.abs(np.minimum(t, 6.0)[..., None] - LEVELS).argmin(axis=-1)
    code = np.where((b < 0) & (code > 0), code + 8, code)
    return code.reshape(n, ncol).astype(np.uint8), e.astype(np.uint8)


def code_values(code, e):
    """f64 values of codes [.., ncol] at exponents [.., ncol / 32]"""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * np.repeat(np.exp2(e.astype(np.float64) - 127), 32, axis=-1)


def as_blocks(code, e):
    n, ncol = code.shape
    c = code.reshape(n, ncol // 32, 2, 16)
    return np.concatenate((e[..., None], c[:, :, 0] | (c[:, :, 1] << 4)), axis=2).reshape(n, -1).astype(np.uint8)


def from_rows(data, n, ncol):
    """(codes, exponents, whether the padding is zero) of MXFP4 rows' bytes"""
    npad = (ncol + 511) // 512 * 512
    c = data[:n * npad // 2].reshape(n, npad // 2)
    s = data[n * npad // 2:].reshape(npad // 512, n, 4, 4).transpose(1, 0, 3, 2).reshape(n, npad // 32)
    return unpadded(np.stack((c & 15, c >> 4), axis=2).reshape(n, npad), s, n, ncol)


def from_tiles(data, nmat, nrow, ncol):
    """the same of matrices laid out in tiles, their rows one after the other"""
    npad, strips = (ncol + 511) // 512 * 512, (nrow + 15) // 16
    size = nmat * strips * 8 * npad
    c = data[:size].reshape(nmat * strips, npad // 128, 4, 16, 16).transpose(0, 3, 1, 2, 4).reshape(-1, npad // 2)
    s = data[size:].reshape(nmat * strips, npad // 512, 4, 16, 4).transpose(0, 3, 1, 4, 2).reshape(-1, npad // 32)
    c = np.stack((c & 15, c >> 4), axis=2).reshape(nmat, strips * 16, npad)
    s = s.reshape(nmat, strips * 16, npad // 32)
    codes, e, clean = unpadded(c[:, :nrow].reshape(-1, npad), s[:, :nrow].reshape(-1, npad // 32), nmat * nrow, ncol)
    return codes, e, clean and not c[:, nrow:].any() and not s[:, nrow:].any()


def unpadded(codes, s, n, ncol):
    return codes[:, :ncol], s[:, :ncol // 32], not codes[:, ncol:].any() and not s[:, ncol // 32:].any()


def random_weights(rng, nmat, ne1, ne0, lo=115, hi=127):
    code = rng.integers(0, 16, (nmat * ne1, ne0)).astype(np.uint8)
    e = rng.integers(lo, hi, (nmat * ne1, ne0 // 32)).astype(np.uint8)
    return code, e


def packed_weights(ex, gq, code, e, nmat):
    torch = torch_()
    blocks = torch.from_numpy(as_blocks(code, e)).cuda()
    return ex.pack(gq, blocks, nmat, code.shape[0] // nmat, code.shape[1])


def rows_of(rng, n, ncol, name, scale=1.0):
    torch = torch_()
    return torch.from_numpy((scale * rng.standard_t(4, (n, ncol))).astype(np.float32)).to(dtype(name)).cuda()


def f64(t):
    return t.double().cpu().numpy()


OUT_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def close_product(got, x, w, out, up=None):
    """y of rows x [m, k] and weights w [n, k] within the bound above"""
    k = x.shape[1]
    unit = (k + 8) * 2.0 ** -23
    y, dy = x @ w.T, unit * (np.abs(x) @ np.abs(w).T)
    if up is not None:
        u, du = x @ up.T, unit * (np.abs(x) @ np.abs(up).T)
        s = y / (1 + np.exp(-y))
        # the slope of silu is at most 1.1; the products' and silu's own roundings are 16 units of the result
        y, dy = s * u, 1.1 * dy * (np.abs(u) + du) + np.abs(s) * du + 16 * 2.0 ** -24 * np.abs(s * u)
    tol = dy + (np.abs(y) + dy) * OUT_UNIT[out] + (2.0 ** -25 if out == "f16" else 1e-44)
    bad = np.abs(got - y) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - y)[bad][:4], tol[bad][:4])


# ---------------------------------------------------------------- rounding
def edge_rows(rng, ncol):
    """every kind of block: normal, ties, zeros, one value, tiny, huge, the largest a hair under a power of two"""
    x = (rng.standard_normal((14, ncol)) * 0.02).astype(np.float32)
    x[1] = np.tile(np.array([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2, -0.25, -0.75, -5.0, 0.0, -0.0, 6.0, 7.9],
                            dtype=np.float32), ncol // 16)
    x[2] = 0
    x[3] = -0.0
    x[4] = 0
    x[4, ::32] = -3e-5
    x[5] *= 1e-37
    x[6] *= 2.0 ** -140
    x[7] = np.float32(3.4028235e38) * np.sign(x[7])
    x[8] *= 1e38
    x[9, ::32] = np.float32(np.nextafter(np.float32(1.0), np.float32(0)))
    x[10] = np.float32(1.4e-45)
    x[11] = 1.0
    x[12, 5::32] = np.nextafter(np.float32(0.02), np.float32(1))
    x[13] = np.round(x[13] / 0.005) * 0.005
    return x


@pytest.mark.parametrize("form", ["blocks", "rows", "tiles"])
@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ncol", [32, 96, 512, 544, 1760])
def test_quantize_matches_the_nearest_levels(gq, ex, src, ncol, form):
    torch = torch_()
    x = torch.from_numpy(edge_rows(np.random.default_rng(ncol), ncol)).to(dtype(src))
    x = torch.nan_to_num(x, posinf=6e4, neginf=-6e4) if src == "f16" else x
    x = torch.nan_to_num(x, posinf=3e38, neginf=-3e38) if src == "bf16" else x
    code, e = round_blocks(x.double().numpy())
    d = x.cuda()
    if form == "rows":
        p, values = ex.quantize(gq, d, values=True)
        c, s, clean = from_rows(p.data.cpu().numpy(), len(x), ncol)
        assert clean and np.array_equal(c, code) and np.array_equal(s, e)
    elif form == "tiles":
        p, values = ex.quantize_weights(gq, d.view(2, 7, ncol), values=True)
        c, s, clean = from_tiles(p.data.cpu().numpy(), 2, 7, ncol)
        assert clean and np.array_equal(c, code) and np.array_equal(s, e)
        values = values.view(14, ncol)
    else:
        blocks, values = ex.quantize_blocks(gq, d, values=True)
        assert np.array_equal(blocks.cpu().numpy(), as_blocks(code, e))
    assert np.array_equal(f64(values), code_values(code, e))


@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_quantize_takes_strided_rows_and_many_blocks(gq, ex, src):
    """rows inside a wider tensor, more blocks than one workgroup, a ragged last one, nothing written past the end"""
    torch = torch_()
    wide = rows_of(np.random.default_rng(3), 77, 3 * 736, src, 0.02)
    x = wide[:, 736:2 * 736]
    code, e = round_blocks(f64(x))
    blocks, values = ex.quantize_blocks(gq, x, values=True)
    assert np.array_equal(blocks.cpu().numpy(), as_blocks(code, e))
    assert np.array_equal(f64(values), code_values(code, e))
    size = 77 * 23 * 17
    out = torch.full((size + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    got = gq.gpuq_mxfp4_quantize_dev(F32 if src == "f32" else BF16, x.data_ptr(), 7, 11, 736, 3 * 736, 0,
                                     out.data_ptr(), None, torch.cuda.current_stream().cuda_stream)
    assert got == size and np.array_equal(out[:size].cpu().numpy(), as_blocks(code, e).ravel())
    assert bool((out[size:] == 0xA5).all())


@pytest.mark.parametrize("src", ["f16", "bf16"])
def test_quantize_every_16_bit_value(gq, ex, src):
    """every finite pattern, in blocks whose largest value puts the scale at 2^0, 2^-2 and 2^-9"""
    torch = torch_()
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(dtype(src)).float()
    for top in (4.0, 1.75, 0.0078125):
        x = torch.where(torch.isfinite(v) & (v.abs() <= top), v, 0.0)
        x = torch.cat((torch.full((len(x) // 31 + 1, 1), top), torch.nn.functional.pad(x, (0, 31 - len(x) % 31)).view(-1, 31)), 1)
        x = x.to(dtype(src))
        code, e = round_blocks(x.double().numpy())
        assert np.array_equal(ex.quantize_blocks(gq, x.cuda()).cpu().numpy(), as_blocks(code, e))


def test_quantize_beside_every_tie(gq, ex):
    """F32 values at, a unit above and a unit below each tie and level, at several scales"""
    torch = torch_()
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=np.float32)
    v = np.concatenate([s * np.concatenate((mid, np.nextafter(mid, np.float32(9)), np.nextafter(mid, np.float32(0))))
                        for s in (np.float32(1), np.float32(-1))])
    v = np.pad(v, (0, 93 - len(v))).reshape(3, 31)
    rows = np.concatenate([np.concatenate((np.full((3, 1), 7.5, np.float32), v), axis=1) * np.float32(2.0 ** k)
                           for k in (0, -6, 20, -120, 120)])
    code, e = round_blocks(rows.astype(np.float64))
    assert np.array_equal(ex.quantize_blocks(gq, torch.from_numpy(rows).cuda()).cpu().numpy(), as_blocks(code, e))


def test_quantize_of_nan_and_infinity(gq, ex):
    torch = torch_()
    x = torch.zeros(4, 64)
    x[0, 3], x[0, 4], x[0, 5] = float("nan"), 2.0, -1.0
    x[1, :32] = float("nan")
    x[2, 0], x[2, 1], x[2, 2] = float("inf"), float("-inf"), 1e30
    x[3, 40], x[3, 41] = float("nan"), float("-inf")
    code, e = round_blocks(x.double().numpy())
    assert code[0, 3] == 0 and e[2, 0] == 252 and code[2, 0] == 7 and code[2, 1] == 15
    for src in ("f32", "bf16"):
        blocks = ex.quantize_blocks(gq, x.to(dtype(src)).cuda())
        assert np.array_equal(blocks.cpu().numpy(), as_blocks(code, e))


def test_blocks_read_back_as_the_library_reads_them(gq, ex):
    """gpuq_dequantize_src_dev, the library's reader of stored MXFP4, gives the rounded values"""
    torch = torch_()
    x = rows_of(np.random.default_rng(5), 64, 2304, "bf16", 0.02)
    blocks, values = ex.quantize_blocks(gq, x, values=True)
    back = torch.empty(64, 2304, device="cuda")
    got = gq.gpuq_dequantize_src_dev(MXFP4, blocks.data_ptr(), back.data_ptr(), back.numel(),
                                     torch.cuda.current_stream().cuda_stream)
    assert got == back.numel() * 4 and torch.equal(back, values.float())


@pytest.mark.parametrize("ne0", [32, 480, 512, 2080])
def test_pack_keeps_every_bit(gq, ex, ne0):
    code, e = random_weights(np.random.default_rng(ne0), 3, 37, ne0, 0, 256)
    p = packed_weights(ex, gq, code, e, 3)
    c, s, clean = from_tiles(p.data.cpu().numpy(), 3, 37, ne0)
    assert clean and np.array_equal(c, code) and np.array_equal(s, e)
    blocks = torch_().from_numpy(as_blocks(code, e)).cuda()
    size = gq.gpuq_mxfp4_bytes(1, 3, 37, ne0)
    out = torch_().empty(size, dtype=torch_().uint8, device="cuda")
    assert gq.gpuq_mxfp4_quantize_dev(MXFP4, blocks.data_ptr(), 3, 37, ne0, ne0, 1, out.data_ptr(), None,
                                      torch_().cuda.current_stream().cuda_stream) == size
    c, s, clean = from_rows(out.cpu().numpy(), 3 * 37, ne0)
    assert clean and np.array_equal(c, code) and np.array_equal(s, e)


# ---------------------------------------------------------------- products
def product_case(gq, ex, x, m, ne1, ne0, out, seed, glu=False):
    rng = np.random.default_rng(seed)
    code, e = random_weights(rng, 1, ne1, ne0)
    w = packed_weights(ex, gq, code, e, 1)
    up = upv = None
    if glu:
        uc, ue = random_weights(rng, 1, ne1, ne0)
        up, upv = packed_weights(ex, gq, uc, ue, 1), code_values(uc, ue)
    if x == "mxfp4":
        rows, values = ex.quantize(gq, rows_of(rng, m, ne0, "bf16", 0.1), values=True)
        xv = f64(values)
    else:
        rows = rows_of(rng, m, ne0, x, 0.1)
        xv = f64(rows)
    y = ex.matmul(gq, rows, w, up=up, out_dtype=dtype(out))
    assert y.dtype == dtype(out) and tuple(y.shape) == (m, ne1)
    close_product(f64(y), xv, code_values(code, e), out, upv)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16", "mxfp4"])
@pytest.mark.parametrize("m,ne1,ne0", [(1, 16, 32), (1, 2048, 1536), (2, 1, 64), (15, 33, 160), (17, 48, 544),
                                       (40, 130, 96), (64, 257, 2304), (65, 129, 32), (129, 64, 640), (200, 300, 1184),
                                       (255, 17, 512), (300, 520, 416), (513, 257, 1024)])
def test_matmul_of_ragged_sizes(gq, ex, x, m, ne1, ne0):
    product_case(gq, ex, x, m, ne1, ne0, "f32", m + ne1)


@pytest.mark.parametrize("x", ["bf16", "mxfp4"])
@pytest.mark.parametrize("out", ["f16", "bf16"])
@pytest.mark.parametrize("m,ne1,ne0", [(3, 36, 256), (33, 50, 128), (150, 260, 288)])
def test_matmul_output_types(gq, ex, x, out, m, ne1, ne0):
    product_case(gq, ex, x, m, ne1, ne0, out, m)


@pytest.mark.parametrize("x", ["f32", "bf16", "mxfp4"])
@pytest.mark.parametrize("m,ne1,ne0", [(1, 40, 96), (20, 70, 256), (90, 65, 544), (300, 200, 320)])
def test_matmul_with_swiglu(gq, ex, x, m, ne1, ne0):
    product_case(gq, ex, x, m, ne1, ne0, "f32", m, glu=True)


@pytest.mark.parametrize("x", ["f32", "f16"])
def test_matmul_keeps_every_bit_of_wide_rows(gq, ex, x):
    """one nonzero term an output: f32 products of the row's value and a power of two are exact"""
    torch = torch_()
    rng = np.random.default_rng(9)
    ne0 = 128
    rows = torch.zeros(32, ne0)
    rows[torch.arange(32), torch.arange(32) * 4] = torch.from_numpy(rng.standard_normal(32).astype(np.float32))
    rows = rows.to(dtype(x)).cuda()
    code = np.full((16, ne0), 2, dtype=np.uint8)
    e = np.full((16, ne0 // 32), 125, dtype=np.uint8)
    y = ex.matmul(gq, rows, packed_weights(ex, gq, code, e, 1))
    want = f64(rows).sum(axis=1, keepdims=True) * 0.25
    assert np.array_equal(f64(y), np.broadcast_to(want, (32, 16)))


@pytest.mark.parametrize("m", [2, 40, 300])
def test_matmul_of_strided_rows_on_another_stream(gq, ex, m):
    torch = torch_()
    rng = np.random.default_rng(m)
    code, e = random_weights(rng, 1, 96, 320)
    w = packed_weights(ex, gq, code, e, 1)
    wide = rows_of(rng, m, 960, "bf16")
    x = wide[:, 320:640]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = ex.matmul(gq, x, w)
    s.synchronize()
    close_product(f64(y), f64(x), code_values(code, e), "f32")


@pytest.mark.parametrize("m", [1, 48, 256])
@pytest.mark.parametrize("x", ["bf16", "mxfp4"])
def test_matmul_of_nan_infinity_and_extreme_scales(gq, ex, m, x):
    """NaN and infinite rows stay their rows' own; a scale of 255 is NaN; the smallest scales still count, the
    largest overflow as f32 does"""
    torch = torch_()
    code, e = np.full((40, 64), 2, dtype=np.uint8), np.full((40, 2), 127, dtype=np.uint8)
    e[3, 0] = 255
    e[4] = 0
    e[5] = 250
    w = packed_weights(ex, gq, code, e, 1)
    v = torch.ones(m, 64)
    if x == "mxfp4":
        rows = ex.quantize(gq, v.cuda())
    else:
        v[0, 1] = float("inf")
        if m > 1:
            v[1, 40] = float("nan")
        rows = v.to(torch.bfloat16).cuda()
    y = f64(ex.matmul(gq, rows, w))
    assert np.isnan(y[:, 3]).all()
    plain = [r for r in range(m) if x == "mxfp4" or r > 1]
    cols = [c for c in range(40) if c not in (3, 4, 5)]
    assert np.array_equal(y[np.ix_(plain, cols)], np.full((len(plain), len(cols)), 64.0))
    assert np.array_equal(y[plain, 4], np.full(len(plain), 64 * 2.0 ** -127))
    assert np.isposinf(y[plain, 5]).all()                # 64 * 2^123, past what f32 holds
    if x == "bf16":
        assert np.isinf(y[0, cols]).all()
        if m > 1:
            assert np.isnan(y[1, cols]).all()


def grouped(rng, counts, ntok, missing=0):
    """(offsets, rows) as numpy for groups of the given sizes, rows at random, `missing` places that no group has"""
    offsets = np.concatenate(([0], np.cumsum(counts))).astype(np.int32)
    rows = rng.integers(0, ntok, offsets[-1] + missing).astype(np.int32)
    rows[offsets[-1]:] = -1
    return offsets, rows


GROUPS = {"step": [0, 1, 0, 0, 2, 1, 0, 1], "few": [3, 0, 17, 16, 0, 1, 33, 5], "chunk": [0, 130, 64, 1, 200, 0, 257, 90],
          "one": [0, 0, 700, 0], "none": [0, 0, 0, 0, 0], "many": [1] * 70 + [0] * 60 + [40]}


@pytest.mark.parametrize("x", ["bf16", "f16", "f32", "mxfp4"])
@pytest.mark.parametrize("name", sorted(GROUPS))
@pytest.mark.parametrize("glu", [False, True], ids=["plain", "glu"])
def test_grouped_products(gq, ex, x, name, glu):
    torch = torch_()
    rng = np.random.default_rng(len(name))
    counts, ne1, ne0, ntok = GROUPS[name], 70, 288, 150
    nmat = len(counts)
    offsets, rows = grouped(rng, counts, ntok, missing=21)
    if len(rows) > 40:
        rows[[5, 30]] = [-1, ntok]                       # rows that name no row of x: zeros
    code, e = random_weights(rng, nmat, ne1, ne0)
    w, wv = packed_weights(ex, gq, code, e, nmat), code_values(code, e).reshape(nmat, ne1, ne0)
    up = None
    if glu:
        uc, ue = random_weights(rng, nmat, ne1, ne0)
        up, upv = packed_weights(ex, gq, uc, ue, nmat), code_values(uc, ue).reshape(nmat, ne1, ne0)
    if x == "mxfp4":
        xr, values = ex.quantize(gq, rows_of(rng, ntok, ne0, "bf16", 0.1), values=True)
        xv = f64(values)
    else:
        xr = rows_of(rng, ntok, ne0, x, 0.1)
        xv = f64(xr)
    g = ex.Group(torch.from_numpy(offsets).cuda(), torch.from_numpy(rows).cuda(), None)
    y = f64(ex.matmul(gq, xr, w, group=g, up=up))
    used = [r for r in range(len(rows)) if 0 <= rows[r] < ntok and r < offsets[-1]]
    assert not y[[r for r in range(len(rows)) if r not in set(used)]].any()
    for m in range(nmat):
        rs = [r for r in used if offsets[m] <= r < offsets[m + 1]]
        if rs:
            close_product(y[rs], xv[rows[rs]], wv[m], "f32", upv[m] if glu else None)


def test_products_past_32_bits(gq, ex):
    """a stack of more than 4 GiB of codes, used at its far end, and rows of x past 4 GiB"""
    torch = torch_()
    nmat, ne1, ne0 = 640, 2048, 7168
    rng = np.random.default_rng(0)
    code, e = random_weights(rng, 1, ne1, ne0)
    one = torch.from_numpy(as_blocks(code, e)).cuda()
    size = gq.gpuq_mxfp4_bytes(2, nmat, ne1, ne0)
    assert size > 1 << 32
    data = torch.zeros(size, dtype=torch.uint8, device="cuda")
    p = ex.pack(gq, one, 1, ne1, ne0).data
    nc = ne1 * ne0 // 2
    data[(nmat - 1) * nc:nmat * nc] = p[:nc]
    data[size - ne1 * ne0 // 32:] = p[nc:]
    w = ex.Packed(data, nmat, ne1, ne0)
    nx = (1 << 32) // (ne0 * 2) + 200
    x = torch.zeros(nx, ne0, dtype=torch.bfloat16, device="cuda")
    x[-300:] = rows_of(rng, 300, ne0, "bf16", 0.1)
    wv, xv = code_values(code, e), f64(x[-300:])
    for n in (3, 300):
        counts = torch.zeros(nmat + 1, dtype=torch.int32, device="cuda")
        counts[-1] = n
        rows = torch.arange(nx - n, nx, dtype=torch.int32, device="cuda")
        y = ex.matmul(gq, x, w, group=ex.Group(counts, rows, None))
        close_product(f64(y)[:, :64], xv[300 - n:], wv[:64], "f32")
    many = torch.cat((rows[:1].expand(nmat * 300 - 300), rows))          # enough rows a group for whole tiles
    counts[-1] = many.numel()
    y = ex.matmul(gq, x, w, group=ex.Group(counts, many.contiguous(), None), out_dtype=torch.bfloat16)
    close_product(f64(y[-300:])[:, :64], xv, wv[:64], "bf16")


# ---------------------------------------------------------------- routing
def check_choice(ids, weights, logits, k, score, bias, ngroup, keep, renorm, scale):
    """a choice against f64 scores: ids in the order of their keys up to 32 units, nothing better left out"""
    unit = 32 * 2.0 ** -24
    x = logits.astype(np.float64)
    n, nexp = x.shape
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-x)) if score == "sigmoid" else np.exp(x - x.max(axis=1, keepdims=True))
    if score == "softmax":
        s /= s.sum(axis=1, keepdims=True)
    by_logit = bias is None and ngroup == 1
    key = x if by_logit else s + (0 if bias is None else bias.astype(np.float64))
    for t in range(n):
        kt = key[t].copy()
        slack = 0 if by_logit else unit * (1 + np.abs(kt).max())
        if ngroup > 1:
            parts = np.sort(kt.reshape(ngroup, -1), axis=1)[:, -2:].sum(axis=1)
            used = set((ids[t] // (nexp // ngroup)).tolist())
            assert len(used) <= keep
            order = np.sort(parts)[::-1]
            assert all(parts[g] >= order[keep - 1] - 2 * slack for g in used)
            kept = [g for g in range(ngroup) if parts[g] > order[keep - 1] + 2 * slack or g in used]
            if len(kept) < keep:
                kept = [g for g in range(ngroup) if parts[g] >= order[keep - 1]]
            mask = np.ones(ngroup, bool)
            mask[kept] = False
            kt.reshape(ngroup, -1)[mask] = -np.inf
        chosen = ids[t]
        assert len(set(chosen.tolist())) == k and ((chosen >= 0) & (chosen < nexp)).all()
        kc = kt[chosen]
        assert (kc[:-1] >= kc[1:] - slack).all()
        rest = np.delete(kt, chosen)
        assert not len(rest) or kc.min() >= rest.max() - slack
        if slack == 0:      # exact order, ties at the lowest index
            assert chosen.tolist() == np.argsort(-kt, kind="stable")[:k].tolist()
        w = s[t][chosen] / (s[t][chosen].sum() if renorm else 1) * scale
        np.testing.assert_allclose(weights[t], w, rtol=unit, atol=1e-37)


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ntok,nexp,k,ngroup,keep", [(1, 8, 2, 1, 1), (5, 1, 1, 1, 1), (7, 64, 6, 1, 1), (130, 100, 8, 1, 1),
                                                     (33, 256, 8, 8, 4), (9, 160, 6, 8, 3), (6, 384, 8, 1, 1), (70, 384, 16, 1, 1),
                                                     (9, 300, 17, 4, 3), (9, 640, 4, 32, 9),
                                                     (2049, 8, 2, 1, 1), (2100, 256, 8, 8, 4), (2050, 100, 7, 1, 1),
                                                     (2053, 480, 16, 16, 5), (2051, 384, 1, 4, 1), (2050, 36, 4, 12, 5),
                                                     (3, 512, 10, 4, 2), (3, 1000, 64, 1, 1), (4, 24, 4, 12, 5)])
def test_route(gq, ex, src, ntok, nexp, k, ngroup, keep):
    torch = torch_()
    rng = np.random.default_rng(nexp)
    logits = torch.from_numpy((1.5 * rng.standard_normal((ntok, nexp))).astype(np.float32)).to(dtype(src))
    bias = (0.1 * rng.standard_normal(nexp)).astype(np.float32)
    for score in ("softmax", "sigmoid"):
        for b, renorm, scale in ((None, True, 1.0), (bias, False, 2.5), (bias, True, 1.0)):
            ids, w = ex.route(gq, logits.cuda(), k, score=score, bias=None if b is None else torch.from_numpy(b).cuda(),
                              ngroup=ngroup, keep=keep, renorm=renorm, scale=scale)
            check_choice(ids.cpu().numpy(), w.cpu().numpy(), logits.float().numpy(), k, score, b, ngroup, keep, renorm, scale)


def test_route_ties_and_strides(gq, ex):
    torch = torch_()
    wide = torch.zeros(6, 500, device="cuda")
    wide[:, 300:400] = torch.randint(0, 3, (6, 100), generator=torch.Generator().manual_seed(1)).float().cuda()
    logits = wide[:, 300:400]
    ids, w = ex.route(gq, logits, 9)
    check_choice(ids.cpu().numpy(), w.cpu().numpy(), logits.cpu().numpy(), 9, "softmax", None, 1, 1, True, 1.0)
    ids, _ = ex.route(gq, torch.zeros(3, 64, device="cuda"), 4, score="sigmoid", ngroup=8, keep=2)
    assert ids.cpu().tolist() == [[0, 1, 2, 3]] * 3
    ids, _ = ex.route(gq, torch.zeros(3, 64, device="cuda"), 12, bias=torch.zeros(64, device="cuda"), ngroup=8, keep=2)
    assert ids.cpu().tolist() == [list(range(12))] * 3


@pytest.mark.parametrize("ntok", [8, 2051])
@pytest.mark.parametrize("nexp,k", [(64, 2), (256, 8), (384, 8), (512, 16), (384, 20), (1024, 3)])
def test_route_where_many_reach_the_bound(gq, ex, nexp, k, ntok):
    """keys that rise along the lanes' groups, and rows of few different values: more candidates than there is room for"""
    torch = torch_()
    rng = np.random.default_rng(nexp)
    rows = [np.arange(nexp), -np.arange(nexp), np.arange(nexp) % 16, (np.arange(nexp) % 64 < 8) * 1.0, np.zeros(nexp),
            rng.integers(0, 2, nexp), np.where(np.arange(nexp) % 16 == 3, 1.0, 0.0), np.where(rng.random(nexp) < 0.5, -0.0, 0.0)]
    rows = [rows[i % 8] for i in range(ntok)]
    logits = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    ids, w = ex.route(gq, logits, k)
    want = np.stack([np.argsort(-r.astype(np.float64), kind="stable")[:k] for r in rows])
    assert np.array_equal(ids.cpu().numpy(), want)
    check_choice(ids[:9].cpu().numpy(), w[:9].cpu().numpy(), logits[:9].cpu().numpy(), k, "softmax", None, 1, 1, True, 1.0)


@pytest.mark.parametrize("times", [1, 400])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True], ids=["plain", "bias"])
def test_route_with_nothing_left(gq, ex, score, with_bias, times):
    """masked experts (minus infinity, NaN) are never taken; a row of them alone gets -1 and 0; infinities count"""
    torch = torch_()
    inf, nan = float("inf"), float("nan")
    logits = torch.tensor([[-inf] * 6, [nan] * 6, [-inf, 2.0, nan, -inf, 1.0, -inf], [0.0, inf, 1.0, 2.0, -inf, nan],
                           [-3.4e38] * 6, [-200.0, -300.0, -250.0, -400.0, -500.0, -600.0]], device="cuda")
    logits = logits.repeat(times, 1)
    bias = torch.zeros(6, device="cuda") if with_bias else None
    ids, w = ex.route(gq, logits, 3, score=score, bias=bias)
    assert torch.equal(ids, ids[:6].repeat(times, 1)) and torch.equal(w, w[:6].repeat(times, 1))
    ids, w = ids[:6].cpu().tolist(), w[:6].cpu().numpy()
    assert ids[0] == ids[1] == [-1, -1, -1] and not w[:2].any()
    assert ids[2] == [1, 4, -1] and w[2, 2] == 0 and abs(w[2].sum() - 1) < 1e-6
    assert ids[3][0] == 1 and np.isfinite(w[3]).all()
    assert ids[4] == [0, 1, 2] and np.isfinite(w[4]).all()
    assert np.isfinite(w[5]).all()
    if not with_bias:
        assert ids[5] == [0, 2, 1]
    ids, w = ex.route(gq, logits[:4, :4].contiguous(), 4, score=score, ngroup=2, keep=1)
    assert ids[0].cpu().tolist() == [-1] * 4 and ids[2].cpu().tolist() == [1, -1, -1, -1]


@pytest.mark.parametrize("n,k,nexp", [(1, 1, 1), (1, 8, 256), (3, 5, 7), (257, 8, 384), (2047, 1, 3), (1000, 6, 48),
                                      (9000, 8, 1024), (4096, 2, 1), (1023, 8, 40),
                                      (1025, 8, 40), (150000, 8, 384)])
def test_group(gq, ex, n, k, nexp):
    torch = torch_()
    rng = np.random.default_rng(n)
    ids = rng.integers(-1, nexp, (n, k)).astype(np.int32)
    ids[rng.random((n, k)) < 0.05] = nexp + 3
    if nexp > 8:
        ids[ids == 4] = 5
    g = ex.group(gq, torch.from_numpy(ids).cuda(), nexp)
    flat = ids.ravel()
    on = (flat >= 0) & (flat < nexp)
    order = np.argsort(np.where(on, flat, nexp), kind="stable")
    total = int(on.sum())
    offsets = np.concatenate(([0], np.cumsum(np.bincount(flat[on], minlength=nexp))))
    assert g.offsets.cpu().tolist() == offsets.tolist()
    want = np.where(np.arange(n * k) < total, order, -1)
    assert np.array_equal(g.slots.cpu().numpy(), want)
    assert np.array_equal(g.rows.cpu().numpy(), np.where(want < 0, -1, want // k))


# ---------------------------------------------------------------- graphs, repeats, refusals
def test_a_layer_in_a_graph(gq, ex):
    """route, group, round and multiply captured once and replayed on changing inputs"""
    torch = torch_()
    rng = np.random.default_rng(2)
    nexp, ne1, ne0, ntok = 16, 96, 256, 700
    code, e = random_weights(rng, nexp, ne1, ne0)
    w = packed_weights(ex, gq, code, e, nexp)
    logits, x = rows_of(rng, ntok, nexp, "f32"), rows_of(rng, ntok, ne0, "f32")

    def layer():
        ids, weights = ex.route(gq, logits, 4)
        g = ex.group(gq, ids, nexp)
        return ids, weights, g.rows, ex.matmul(gq, x, w, group=g), ex.matmul(gq, ex.quantize(gq, x), w, group=g, up=w)
    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = layer()
    for seed in range(4):
        r = np.random.default_rng(100 + seed)
        logits.copy_(rows_of(r, ntok, nexp, "f32"))
        x.copy_(rows_of(r, ntok, ne0, "f32"))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, layer()):
            assert torch.equal(a, b)


def test_results_repeat(gq, ex):
    torch = torch_()
    rng = np.random.default_rng(4)
    code, e = random_weights(rng, 8, 200, 1056)
    w = packed_weights(ex, gq, code, e, 8)
    for n in (2, 60, 900):
        x = rows_of(rng, n, 1056, "f32")
        ids, _ = ex.route(gq, rows_of(rng, n, 8, "f32"), 2)
        g = ex.group(gq, ids, 8)
        first = ex.matmul(gq, x, w, group=g)
        for _ in range(3):
            assert torch.equal(first, ex.matmul(gq, x, w, group=ex.group(gq, ids, 8)))


def test_refusals(gq, ex):
    torch = torch_()
    st = torch.cuda.current_stream().cuda_stream
    x = torch.zeros(64, 512, dtype=torch.bfloat16, device="cuda")
    out = torch.zeros(1 << 18, dtype=torch.uint8, device="cuda")
    p, o = x.data_ptr(), out.data_ptr()
    q = gq.gpuq_mxfp4_quantize_dev
    good = [BF16, p, 2, 2, 512, 512, 0, o, None, st]
    assert q(*good) == 4 * 16 * 17
    for at, bad in ((0, Q8_0), (0, MXFP4), (1, None), (1, p + 2), (2, 0), (3, 0), (3, -1), (4, 500), (4, 0), (5, 480),
                    (5, 516), (6, 3), (6, -1), (7, None), (7, o + 1), (8, o + 4)):
        args = list(good)
        args[at] = bad
        assert q(*args) == 0, (at, bad)
    assert q(MXFP4, p, 2, 2, 512, 544, 1, o, None, st) == 0
    assert gq.gpuq_mxfp4_bytes(1, 1, 1, 33) == 0 and gq.gpuq_mxfp4_bytes(2, 1, 0, 32) == 0
    assert gq.gpuq_mxfp4_bytes(1, 1, 3, 544) == 3 * 1024 * 17 // 32 and gq.gpuq_mxfp4_bytes(2, 2, 17, 32) == 64 * 272
    mm = gq.gpuq_mxfp4_matmul_dev
    good = [BF16, p, 64, 512, o, None, 1, 32, 512, None, None, 64, F32, o, None, st]
    for at, bad in ((0, Q8_0), (1, None), (1, p + 2), (2, 0), (3, 500), (4, None), (4, o + 8), (5, o + 8), (6, 0), (6, 2),
                    (6, 70000), (7, 0), (8, 500), (9, o + 2), (10, o + 2), (11, 0), (11, 65), (12, Q8_0), (12, MXFP4),
                    (13, None), (13, o + 4)):
        args = list(good)
        args[at] = bad
        assert mm(*args) == 0, (at, bad)
    assert mm(F32, p, 32, 512, o, None, 1, 32, 512, None, None, 32, F32, o, None, st) == 0      # no scratch
    r = gq.gpuq_route_dev
    assert r(F32, p, 4, 64, 64, 2, 0, None, 1, 1, 1, 1.0, o, o + 1024, st) == 0
    good = [F32, p, 4, 64, 64, 2, 0, None, 1, 1, 1, 1.0, o, o + 1024, st]
    for at, bad in ((0, MXFP4), (1, None), (1, p + 2), (2, 0), (3, 63), (4, 0), (4, 2000), (5, 0), (5, 65), (7, o + 2), (8, 0),
                    (8, 3), (9, 0), (9, 2), (12, None), (12, o + 2), (13, None)):
        args = list(good)
        args[at] = bad
        assert r(*args) == 1, (at, bad)
    g = gq.gpuq_route_group_dev
    assert g(o, 0, 2, 8, o, o, o, None, st) == 1 and g(o, 4, 2, 2000, o, o, o, None, st) == 1
    assert g(o, 8192, 2, 8, o, o, o, None, st) == 1             # needs scratch
    w = ex.Packed(out, 1, 32, 480)
    for call in (lambda: ex.matmul(gq, x, w), lambda: ex.quantize(gq, x[:, :40]), lambda: ex.quantize(gq, x.t()),
                 lambda: ex.quantize(gq, x.cpu()), lambda: ex.route(gq, x, 3, score="other"),
                 lambda: ex.route(gq, x, 513), lambda: ex.pack(gq, out, 1, 32, 480),
                 lambda: ex.group(gq, torch.zeros(4, 2, dtype=torch.int64, device="cuda"), 4)):
        with pytest.raises(ValueError):
            call()
    torch.cuda.synchronize()


def test_a_matrix_of_other_bytes_is_refused(gq, ex):
    torch = torch_()
    x = torch.zeros(4, 512, dtype=torch.bfloat16, device="cuda")
    data = torch.zeros(32 * 512 // 32 * 17, dtype=torch.uint8, device="cuda")
    good, rows = ex.Packed(data, 1, 32, 512), ex.quantize(gq, x)
    assert not ex.matmul(gq, x, good).any() and not ex.matmul(gq, rows, good, up=good).any()
    short = good._replace(data=data[:-16])
    for call in (lambda: ex.matmul(gq, x, short), lambda: ex.matmul(gq, x, good, up=short),
                 lambda: ex.matmul(gq, x, good._replace(nmat=2), group=ex.Group(torch.zeros(3, dtype=torch.int32, device="cuda"),
                                                                                torch.zeros(4, dtype=torch.int32, device="cuda"), None)),
                 lambda: ex.matmul(gq, rows._replace(n=5), good)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
def test_many_rows_round_as_few_do(gq, ex, src):
    """more rows than the caches hold take loads and stores of their own kind"""
    torch = torch_()
    n, ncol = (129 << 20) // (512 * (4 if src == "f32" else 2)) + 3, 512
    torch.manual_seed(7)
    x = torch.randn(n, ncol, device="cuda").to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[src])
    x[n // 3] = float("inf")
    x[n // 3 + 1, ::7] = float("nan")
    blocks, values = ex.quantize_blocks(gq, x, values=True)
    for a in range(0, n, n // 3):
        b, v = ex.quantize_blocks(gq, x[a:a + n // 3], values=True)
        assert torch.equal(blocks[a:a + n // 3], b) and torch.equal(values[a:a + n // 3], v)

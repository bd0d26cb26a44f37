"""The 4-bit operators against their definition in 64 bits (tests/fp4_reference.py), at the sizes and values where they
can go wrong: ragged rows and columns, tiles that end inside a block, odd pitches, every code with every factor, ties,
zero, tiny and huge blocks, blocks that are not finite, residuals in place, captured and replayed calls."""
import numpy as np
import pytest
import torch

import fp4_reference as ref

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
# what a result below the type's normal range may be off by on top: half of its smallest step
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _dt(fx, name):
    return {"f32": fx.F32, "f16": fx.F16, "bf16": fx.BF16}[name]


class Matrix:
    """Device buffers of a 4-bit matrix, with a guard behind each that must survive."""

    def __init__(self, fx, rows, cols, fmt, scale=1.0, packed=None):
        self.nc, self.ns = fx.fp4_bytes(rows, cols, fmt)
        self.rows, self.cols, self.fmt = rows, cols, fmt
        self.codes = torch.full((self.nc + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        self.scales = torch.full((self.ns + 64,), 0xA5, dtype=torch.uint8, device="cuda")
        if packed is not None:
            self.codes[:self.nc] = torch.from_numpy(packed[0].reshape(-1)).cuda()
            self.scales[:self.ns] = torch.from_numpy(packed[1]).cuda()
        self.h = fx.Fp4(self.codes.data_ptr(), self.scales.data_ptr(), rows, cols, fmt, scale)

    def read(self):
        assert (self.codes[self.nc:] == 0xA5).all() and (self.scales[self.ns:] == 0xA5).all()
        return ref.unpack(self.codes[:self.nc].cpu().numpy(), self.scales[:self.ns].cpu().numpy(), self.rows, self.cols,
                          self.fmt)


def _random_matrix(fx, rng, rows, cols, fmt, std=1.0, scale=1.0):
    code, byte = ref.quantize(rng.standard_normal((rows, cols)) * std, fmt)
    return Matrix(fx, rows, cols, fmt, scale, ref.pack(code, byte)), ref.values(code, byte, fmt, scale)


def _plain(x, name, ld):
    """x (float64 numpy) on the device in the given type with row pitch ld, and what that type made of it."""
    wide = torch.full((max(1, x.shape[0]), ld), 7.0, dtype=TORCH[name])
    wide[:x.shape[0], :x.shape[1]] = torch.from_numpy(x).to(TORCH[name])
    return wide.cuda(), wide[:x.shape[0], :x.shape[1]].double().numpy()


def _inputs(rng, rows, cols, fmt, name):
    """Normal values with blocks that are zero, tiny, huge and full of ties."""
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-3, 4, (rows, 1)))
    for i in range(0, rows * -(-cols // fmt), 3):
        r, b = i % rows, (i // rows) % -(-cols // fmt)
        blk = x[r, b * fmt:(b + 1) * fmt]
        kind = (i // 3) % 5
        if kind == 0:
            blk[:] = 0
        elif kind == 1:
            blk *= 2.0 ** (-14 if name == "f16" else -40)
        elif kind == 2:
            blk *= 2.0 ** (10 if name == "f16" else 40)
        elif kind == 3:  # every value a border between two codes, for a factor of 2
            blk[:] = rng.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], blk.shape) * rng.choice([-2, 2], blk.shape)
            blk[0] = 12.0
        else:  # a maximum whose sixth lies between two factors
            blk[0] = 6 * (1 + (2 * rng.integers(0, 8) + 1) / 16)
    return x


SIZES = [(1, 1, 0), (1, 16, 3), (2, 2560, 0), (3, 31, 1), (17, 33, 0), (33, 64, 8), (127, 257, 7), (129, 1000, 0),
         (130, 96, 5), (257, 513, 0)]


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", SIZES)
def test_quantize_is_the_definition(fx, ctx, rows, cols, pad, name, fmt):
    rng = np.random.default_rng(rows * 1000 + cols)
    dev, x = _plain(_inputs(rng, rows, cols, fmt, name), name, cols + pad)
    q = Matrix(fx, rows, cols, fmt)
    torch.cuda.synchronize()
    ctx.fp4_quantize(dev.data_ptr(), _dt(fx, name), cols + pad, q.h)
    ctx.sync()
    code, byte, clean = q.read()
    want, wbyte = ref.quantize(x, fmt)
    assert clean
    assert (byte == wbyte).all()
    # the sign of a zero is free
    assert (ref.values(code, byte, fmt) == ref.values(want, wbyte, fmt)).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("scale", [2.0 ** -20, 0.5, 4.0, 2.0 ** 30])
def test_quantize_divides_by_the_matrix_scale(fx, ctx, scale, fmt):
    rng = np.random.default_rng(5)
    dev, x = _plain(rng.standard_normal((65, 200)) * 100 * scale, "f32", 200)
    q = Matrix(fx, 65, 200, fmt, scale)
    torch.cuda.synchronize()
    ctx.fp4_quantize(dev.data_ptr(), fx.F32, 200, q.h)
    ctx.sync()
    code, byte, clean = q.read()
    want, wbyte = ref.quantize(x, fmt, scale)
    assert clean and (byte == wbyte).all() and (ref.values(code, byte, fmt) == ref.values(want, wbyte, fmt)).all()


@pytest.mark.parametrize("fmt", [16, 32])
def test_quantize_f32_next_to_borders(fx, ctx, fmt):
    """f32 values one unit on either side of every border of the codes, and block maxima one unit on either side of every
    border of the factors."""
    rows = []
    for byte in range(1, 127):
        s = ref.E4M3[byte] if fmt == 16 else 2.0 ** (byte - 60)
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            t = np.float32(border * s)
            r = np.zeros(fmt)
            r[:4] = [6 * s, np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(1e38))]
            rows.append(r)
        if fmt == 16 and byte < 126:
            t = np.float32(6 * (ref.E4M3[byte] + ref.E4M3[byte + 1]) / 2)
            for a in (np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(1e38))):
                rows.append(np.concatenate([[a], np.zeros(fmt - 1)]))
    x = np.array(rows)
    dev, x = _plain(x, "f32", fmt)
    q = Matrix(fx, len(rows), fmt, fmt)
    torch.cuda.synchronize()
    ctx.fp4_quantize(dev.data_ptr(), fx.F32, fmt, q.h)
    ctx.sync()
    code, byte, _ = q.read()
    want, wbyte = ref.quantize(x, fmt)
    assert (byte == wbyte).all() and (code & 7 == want & 7).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_blocks_that_are_not_finite(fx, ctx, name, fmt):
    x = np.random.default_rng(3).standard_normal((40, 100))
    x[0, 0], x[1, 99], x[2, 50], x[39, 17] = np.nan, np.inf, -np.inf, np.nan
    dev, x = _plain(x, name, 100)
    q = Matrix(fx, 40, 100, fmt)
    out = torch.zeros(40, 100, dtype=TORCH[name], device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_quantize(dev.data_ptr(), _dt(fx, name), 100, q.h)
    ctx.fp4_dequantize(q.h, out.data_ptr(), _dt(fx, name), 100)
    ctx.sync()
    code, byte, clean = q.read()
    want, wbyte = ref.quantize(x, fmt)
    assert clean and (byte == wbyte).all()
    v = ref.values(want, wbyte, fmt)
    got = out.double().cpu().numpy()
    assert (np.isnan(got) == np.isnan(v)).all() and np.isnan(v).sum() > 4 * fmt - fmt
    assert (got[~np.isnan(v)] == v[~np.isnan(v)]).all()  # at most six significant bits: exact in every type


def test_extreme_f32_values(fx, ctx):
    """The largest and smallest f32 values, subnormal ones among them: factors at both ends of their range."""
    big = float(np.finfo(np.float32).max)
    x = np.zeros((8, 64))
    x[0], x[1], x[2] = big, -big, 2.0 ** -149
    x[3, ::2], x[4, 1] = 2.0 ** -126, 3e-39
    x[5, 0], x[5, 1] = big, 2.0 ** -149
    x[6], x[7] = 448 * 6.0, 448 * 6.5
    dev, x = _plain(x, "f32", 64)
    for fmt in (16, 32):
        q = Matrix(fx, 8, 64, fmt)
        torch.cuda.synchronize()
        ctx.fp4_quantize(dev.data_ptr(), fx.F32, 64, q.h)
        ctx.sync()
        code, byte, _ = q.read()
        want, wbyte = ref.quantize(x, fmt)
        assert (byte == wbyte).all() and (ref.values(code, byte, fmt) == ref.values(want, wbyte, fmt)).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 0.3, -2.5])
def test_dequantize_every_code_with_every_factor(fx, ctx, scale, name, fmt):
    code = np.tile(np.arange(16), (256, fmt // 16 * 3))
    byte = np.repeat(np.arange(256)[:, None], 3, 1).astype(np.uint8)
    if fmt == 16:
        byte &= 127  # e4m3 factors are not negative
    m = Matrix(fx, 256, code.shape[1], fmt, scale, ref.pack(code, byte))
    out = torch.zeros(256, code.shape[1], dtype=TORCH[name], device="cuda")
    torch.cuda.synchronize()
    ctx.saturated_stores(reset=True)
    ctx.fp4_dequantize(m.h, out.data_ptr(), _dt(fx, name), code.shape[1])
    ctx.sync()
    want = ref.values(code, byte, fmt, float(np.float32(scale)))
    got = out.double().cpu().numpy()
    over = {"f32": float(np.finfo(np.float32).max), "f16": 65504.0, "bf16": float(torch.finfo(torch.bfloat16).max)}[name]
    assert (np.isnan(got) == np.isnan(want)).all()
    fine = np.isfinite(want) & (np.abs(want) <= over)
    # one rounding to f32 (the product with the matrix's scale), one to the type
    tol = (HALF_STEP[name] + 2.0 ** -24) * np.abs(want) + TINY[name] + 2.0 ** -150
    assert (np.abs(got - want)[fine] <= tol[fine]).all()
    beyond = np.isfinite(want) & ~fine & (np.abs(want) > over * (1 + 2 * HALF_STEP[name]))
    if name == "f16":
        assert (np.abs(got[beyond]) == 65504.0).all()
        assert (ctx.saturated_stores(reset=True) > 0) == bool(beyond.any())
    else:
        assert np.isinf(got[beyond]).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,pad", SIZES)
def test_dequantize_sizes_and_pitches(fx, ctx, rows, cols, pad, name, fmt):
    m, want = _random_matrix(fx, np.random.default_rng(rows + cols), rows, cols, fmt)
    out = torch.full((rows + 1, cols + pad), 7.0, dtype=TORCH[name], device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_dequantize(m.h, out.data_ptr(), _dt(fx, name), cols + pad)
    ctx.sync()
    got = out.double().cpu().numpy()
    assert (got[:rows, :cols] == want).all()  # six significant bits
    assert (got[rows:] == 7).all() and (got[:, cols:] == 7).all()


def _product_tolerance(x, w, want, out, gate, residual):
    """f32 sums of exact products: an instruction adds the products of 64 columns to the accumulator, which costs at most a
    truncation of the running sum and one of the aligned products, 2^-23 of the sum of magnitudes each; the parts of a
    split K are added in f32 (at most 8). Then the scale, the gate and the residual, a rounding each (the scales' own
    product is one more), and the output's type."""
    mag = np.abs(x) @ np.abs(w).T
    g = 1.0 if gate is None else np.abs(gate)
    steps = -(-x.shape[1] // 64) + 8
    tol = g * (mag * steps * 2 * 2.0 ** -23 + 3 * 2.0 ** -24 * np.abs(x @ w.T))
    if residual is not None:
        tol = tol + 2.0 ** -24 * np.abs(want)
    return tol + HALF_STEP[out] * np.abs(want) + TINY[out]


def _product(fx, ctx, M, N, K, fmt, out, gated=False, pad=0, in_place=False, scales=(1.0, 1.0), seed=0):
    rng = np.random.default_rng(seed * 7 + M * 31 + N * 17 + K)
    x, xv = _random_matrix(fx, rng, M, K, fmt, scale=scales[0])
    w, wv = _random_matrix(fx, rng, N, K, fmt, std=0.1, scale=scales[1])
    want = xv @ wv.T
    gate = residual = None
    dev = torch.full((M + 1, N + pad), 7.0, dtype=TORCH[out], device="cuda")
    args = {}
    if gated:
        gate = rng.standard_normal(N).astype(np.float32)
        residual = rng.standard_normal((M, N)).astype(np.float32)
        want = residual.astype(np.float64) + gate.astype(np.float64) * want
        g = torch.from_numpy(gate).cuda()
        if in_place:
            dev[:M, :N] = torch.from_numpy(residual).cuda()
            args = dict(gate_ptr=g.data_ptr(), residual_ptr=dev.data_ptr(), ld_residual=N + pad)
        else:
            r = torch.zeros(M, N + 3, device="cuda")
            r[:, :N] = torch.from_numpy(residual).cuda()
            args = dict(gate_ptr=g.data_ptr(), residual_ptr=r.data_ptr(), ld_residual=N + 3)
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, dev.data_ptr(), _dt(fx, out), N + pad, **args)
    ctx.sync()
    got = dev.double().cpu().numpy()
    tol = _product_tolerance(xv, wv, want, out, gate, residual)
    assert (np.abs(got[:M, :N] - want) <= tol).all(), (np.abs(got[:M, :N] - want) / tol).max()
    assert (got[M:] == 7).all() and (got[:, N:] == 7).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("M,N,K", [
    (1, 1, 1), (1, 128, 64), (1, 130, 256), (1, 300, 2560), (2, 127, 31), (7, 129, 1111), (16, 256, 512), (17, 64, 257),
    (33, 128, 300), (64, 384, 1024), (65, 100, 96), (77, 1001, 1111), (128, 128, 256), (129, 257, 640), (200, 640, 1000),
    (256, 256, 2048), (300, 513, 96),
    # low tiles with four and with nine k-slices under way, alone and split
    (12, 2000, 9000), (16, 20000, 600), (24, 500, 6000), (30, 2560, 3000), (20, 19000, 300),
    # enough tiles for pairs of CTAs: ragged in every direction, one and several tiles per pair, many k-slices
    (1290, 2300, 70), (700, 3300, 300), (1025, 2049, 1600), (2600, 5200, 64), (150, 9600, 513)])
def test_product_sizes(fx, ctx, M, N, K, fmt):
    _product(fx, ctx, M, N, K, fmt, "f32")


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("gated,in_place", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("M,N,K,pad", [(3, 200, 500, 0), (100, 131, 260, 5), (140, 256, 3000, 8), (520, 700, 300, 1), (24, 260, 6000, 2), (16, 2560, 2560, 0),
                                       (90, 128, 7000, 3), (1300, 2200, 300, 4),
                                       (1500, 6000, 296, 3)])
def test_product_outputs(fx, ctx, M, N, K, pad, gated, in_place, out):
    if in_place and out != "f32":
        pytest.skip("a residual in place is f32")
    _product(fx, ctx, M, N, K, 16 if K % 8 else 32, out, gated, pad, in_place, scales=(0.5, 1.7), seed=1)


@pytest.mark.parametrize("fmt", [16, 32])
def test_product_rows_of_nan(fx, ctx, fmt):
    """A NaN factor reaches exactly its row of x, or its row of w (a column of the result)."""
    rng = np.random.default_rng(9)
    M, N, K = 130, 140, 300
    cx, bx = ref.quantize(rng.standard_normal((M, K)), fmt)
    cw, bw = ref.quantize(rng.standard_normal((N, K)), fmt)
    nan = 255 if fmt == 32 else 127
    bx[3, 0], bx[129, -1], bw[139, 2] = nan, nan, nan
    x, w = Matrix(fx, M, K, fmt, 1.0, ref.pack(cx, bx)), Matrix(fx, N, K, fmt, 1.0, ref.pack(cw, bw))
    out = torch.zeros(M, N, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, N)
    ctx.sync()
    want = np.zeros((M, N), bool)
    want[[3, 129]] = True
    want[:, 139] = True
    assert (torch.isnan(out).cpu().numpy() == want).all()


def test_product_of_a_row_slice(fx, ctx):
    """Rows [128, ...) of a matrix are a matrix of their own."""
    rng = np.random.default_rng(10)
    w, wv = _random_matrix(fx, rng, 300, 200, 16)
    x, xv = _random_matrix(fx, rng, 20, 200, 16)
    pitch, chunks = 16 * 7, 4
    part = fx.Fp4(w.codes.data_ptr() + 128 * pitch, w.scales.data_ptr() + chunks * 512, 172, 200, 16, 1.0)
    out = torch.zeros(20, 172, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, part, out.data_ptr(), fx.F32, 172)
    ctx.sync()
    want = xv @ wv[128:].T
    assert (np.abs(out.double().cpu().numpy() - want) <= _product_tolerance(xv, wv[128:], want, "f32", None, None)).all()


def _few_row_tolerance(mag, K, xname):
    """f32 sums of exact products: an instruction adds the products of 16 columns and one bf16 part of x to the accumulator,
    at most a truncation of the running sum and one of the aligned products, 2^-23 of the sum of magnitudes each; then at
    most 64 partial sums, and the scale (a rounding, and one for the tests' own use of it)."""
    parts = {"bf16": 1, "f16": 2, "f32": 3}[xname]
    return mag * (2 * parts * -(-K // 16) + 64 + 2) * 2.0 ** -23


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("xname,out", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("M,N,K,pad", [(1, 1, 1, 0), (1, 300, 2560, 0), (2, 129, 1025, 3), (3, 128, 31, 1), (4, 260, 96, 0),
                                       (5, 97, 1000, 0), (8, 64, 2048, 8), (16, 200, 700, 0)])
def test_few_row_product(fx, ctx, M, N, K, pad, xname, out, fmt):
    rng = np.random.default_rng(M + N + K)
    w, wv = _random_matrix(fx, rng, N, K, fmt, std=0.1, scale=0.7)
    dev, x = _plain(rng.standard_normal((M, K)), xname, K + pad)
    got = torch.full((M + 1, N + pad), 7.0, dtype=TORCH[out], device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), _dt(fx, xname), K + pad, M, w.h, got.data_ptr(), _dt(fx, out), N + pad)
    ctx.sync()
    wv = wv / 0.7 * float(np.float32(0.7))
    want = x @ wv.T
    mag = np.abs(x) @ np.abs(wv).T
    tol = _few_row_tolerance(mag, K, xname) + HALF_STEP[out] * np.abs(want) + TINY[out]
    have = got.double().cpu().numpy()
    assert (np.abs(have[:M, :N] - want) <= tol).all()
    assert (have[M:] == 7).all() and (have[:, N:] == 7).all()


@pytest.mark.parametrize("M,K", [(1, 60000), (3, 20000), (16, 30000), (1, 65536), (5, 65536)])
def test_few_row_product_of_long_rows(fx, ctx, M, K):
    """Rows of x that fit shared memory only in parts, or not all at once."""
    rng = np.random.default_rng(K)
    w, wv = _random_matrix(fx, rng, 40, K, 16)
    dev, x = _plain(rng.standard_normal((M, K)), "f32", K)
    out = torch.zeros(M, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), fx.F32, K, M, w.h, out.data_ptr(), fx.F32, 40)
    ctx.sync()
    want = x @ wv.T
    tol = _few_row_tolerance(np.abs(x) @ np.abs(wv).T, K, "f32") + 2.0 ** -24 * np.abs(want)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("N,K", [(2560, 9728), (19000, 300), (9728, 1000), (128, 128)])
def test_few_row_product_of_many_columns(fx, ctx, N, K):
    """Several rounds of weight rows per block, and K split among warps and CTAs."""
    rng = np.random.default_rng(N)
    for M, name in ((1, "bf16"), (4, "f32"), (16, "f16")):
        w, wv = _random_matrix(fx, rng, N, K, 32 if M == 4 else 16, std=0.1)
        dev, x = _plain(rng.standard_normal((M, K)), name, K)
        out = torch.zeros(M, N, device="cuda")
        torch.cuda.synchronize()
        ctx.gemv_fp4(dev.data_ptr(), _dt(fx, name), K, M, w.h, out.data_ptr(), fx.F32, N)
        ctx.sync()
        want = x @ wv.T
        tol = _few_row_tolerance(np.abs(x) @ np.abs(wv).T, K, name) + 2.0 ** -24 * np.abs(want)
        assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("fmt", [16, 32])
def test_few_row_product_with_every_factor(fx, ctx, fmt):
    """Every finite factor with every code, against x that picks out one column: exact products, so exact results (where
    they are normal f32 values). Factors of NaN give NaN in their row."""
    code = np.tile(np.arange(16), (256, fmt // 16))
    byte = np.arange(256).astype(np.uint8)[:, None]
    if fmt == 16:
        byte &= 127
    w = Matrix(fx, 256, fmt, fmt, 1.0, ref.pack(code, byte))
    wv = ref.values(code, byte, fmt)
    for name in ("f32", "f16", "bf16"):
        for first in range(0, fmt, 16):
            x = np.zeros((16, fmt))
            x[np.arange(16), first + np.arange(16)] = {"f32": 1 + 2.0 ** -23, "f16": 1 + 2.0 ** -10, "bf16": 1 + 2.0 ** -7}[name]
            dev, xv = _plain(x, name, fmt)
            out = torch.zeros(16, 256, device="cuda")
            torch.cuda.synchronize()
            ctx.gemv_fp4(dev.data_ptr(), _dt(fx, name), fmt, 16, w.h, out.data_ptr(), fx.F32, 256)
            ctx.sync()
            with np.errstate(over="ignore"):
                want = np.stack([(xv[i, first + i] * wv[:, first + i]) for i in range(16)])
            got = out.double().cpu().numpy()
            # rows of w that hold values beyond the f32 range (factors above 2^125) are left to the formats
            inside = np.isnan(wv).any(1) | (np.abs(wv).max(1) < 3.4e38)
            assert inside.sum() >= 254 - 2
            assert (np.isnan(got) == np.isnan(want))[:, inside].all()
            # parts of x times a weight are exact; adding up to three of them rounds twice
            fine = inside & np.isfinite(want) & (np.abs(want) < 3e38) & ((np.abs(want) > 2.0 ** -100) | (want == 0))
            assert (np.abs(got - want)[fine] <= 2 * 2.0 ** -23 * np.abs(want)[fine]).all()


def test_few_row_product_of_extreme_rows(fx, ctx):
    """Rows of x with infinities, NaN and values at both ends of the f32 range stay rows of their own; a huge value at a
    weight of zero does not cost its neighbours their digits."""
    code = np.zeros((40, 64), np.int64)
    code[:, 1:] = 2  # 1.0, but for column 0
    w = Matrix(fx, 40, 64, 16, 1.0, ref.pack(code, np.full((40, 4), 0x38, np.uint8)))  # factors of 1
    x = np.zeros((6, 64))
    x[0, 0], x[0, 1] = 3e38, 1e-30
    x[1, 1] = float(np.finfo(np.float32).max)
    x[2, 5], x[3, 6] = np.inf, np.nan
    x[4, 0] = np.inf  # times zero
    x[5, 3] = 1.5
    dev, xv = _plain(x, "f32", 64)
    out = torch.zeros(6, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), fx.F32, 64, 6, w.h, out.data_ptr(), fx.F32, 40)
    ctx.sync()
    got = out.double().cpu().numpy()
    assert (np.abs(got[0] - xv[0, 1]) <= 2.0 ** -22 * 1e-30).all()
    assert (np.abs(got[1] / xv[1, 1] - 1) <= 2.0 ** -22).all()
    assert (got[2] == np.inf).all() and np.isnan(got[3]).all() and np.isnan(got[4]).all() and (got[5] == 1.5).all()


def test_nothing_to_do(fx, ctx):
    """No rows: accepted, nothing is written, no memory is needed."""
    m = Matrix(fx, 5, 64, 16)
    none = fx.Fp4(None, None, 0, 64, 16, 1.0)
    out = torch.full((8, 8), 7.0, device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_quantize(None, fx.F32, 64, none)
    ctx.fp4_dequantize(none, None, fx.F32, 64)
    ctx.gemm_fp4(none, m.h, None, fx.F32, 5)
    ctx.gemm_fp4(m.h, none, None, fx.F32, 0)
    ctx.gemv_fp4(None, fx.F32, 64, 0, m.h, None, fx.F32, 5)
    ctx.gemv_fp4(out.data_ptr(), fx.F32, 64, 1, none, None, fx.F32, 0)
    ctx.sync()
    assert (out == 7).all()


def test_saturating_product_is_counted(fx, ctx):
    code, byte = np.full((20, 64), 7), np.full((20, 4), 0x7E, np.uint8)  # 6 * 448 everywhere
    a, b = Matrix(fx, 20, 64, 16, 1.0, ref.pack(code, byte)), Matrix(fx, 20, 64, 16, 1.0, ref.pack(code, byte))
    out = torch.zeros(20, 20, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.sync()
    ctx.saturated_stores(reset=True)
    ctx.gemm_fp4(a.h, b.h, out.data_ptr(), fx.F16, 20)
    ctx.sync()
    assert (out == 65504).all() and ctx.saturated_stores(reset=True) > 0


def _feed_forward(fx, c, x, w1, w2, h_res, gate, bufs, N1, N2, M, K):
    """As a feed-forward block uses them: activations -> 4 bits -> product -> 4 bits -> product onto the residual."""
    c.fp4_quantize(x.data_ptr(), fx.BF16, K, bufs["q1"].h)
    c.gemm_fp4(bufs["q1"].h, w1.h, bufs["mid"].data_ptr(), fx.BF16, N1)
    c.fp4_quantize(bufs["mid"].data_ptr(), fx.BF16, N1, bufs["q2"].h)
    c.gemm_fp4(bufs["q2"].h, w2.h, h_res.data_ptr(), fx.F32, N2, gate_ptr=gate.data_ptr(), residual_ptr=h_res.data_ptr(),
               ld_residual=N2)


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("M", [1, 40, 300])
def test_a_feed_forward_block(fx, ctx, M, fmt):
    """The operators one after another on the context's stream, each step checked against 64 bits from the step before,
    then captured into a graph and replayed twice: the same bits."""
    rng = np.random.default_rng(M)
    K, N1, N2 = 320, 500, 200
    w1, w1v = _random_matrix(fx, rng, N1, K, fmt, std=0.1)
    w2, w2v = _random_matrix(fx, rng, N2, N1, fmt, std=0.1)
    x, xv = _plain(rng.standard_normal((M, K)), "bf16", K)
    res0 = torch.from_numpy(rng.standard_normal((M, N2)).astype(np.float32)).cuda()
    gate = torch.from_numpy(rng.standard_normal(N2).astype(np.float32)).cuda()
    bufs = {"q1": Matrix(fx, M, K, fmt), "q2": Matrix(fx, M, N1, fmt),
            "mid": torch.zeros(M, N1, dtype=torch.bfloat16, device="cuda")}
    res = res0.clone()
    torch.cuda.synchronize()
    _feed_forward(fx, ctx, x, w1, w2, res, gate, bufs, N1, N2, M, K)
    ctx.sync()
    q1 = ref.values(*ref.quantize(xv, fmt), fmt)
    mid = bufs["mid"].double().cpu().numpy()
    assert (np.abs(mid - q1 @ w1v.T) <= _product_tolerance(q1, w1v, q1 @ w1v.T, "bf16", None, None)).all()
    q2 = ref.values(*ref.quantize(mid, fmt), fmt)
    g, r0 = gate.double().cpu().numpy(), res0.double().cpu().numpy()
    want = r0 + g * (q2 @ w2v.T)
    first = res.clone()
    assert (np.abs(first.double().cpu().numpy() - want) <= _product_tolerance(q2, w2v, want, "f32", g, r0)).all()
    stream = torch.cuda.ExternalStream(ctx.stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        _feed_forward(fx, ctx, x, w1, w2, res, gate, bufs, N1, N2, M, K)
    for _ in range(2):
        res.copy_(res0)
        bufs["mid"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.sync()
        assert torch.equal(res, first)


def test_every_operator_captured_and_replayed(fx, ctx):
    """Two graphs of the same calls on different data share nothing; replays give the bits of the eager calls."""
    rng = np.random.default_rng(30)
    stream = torch.cuda.ExternalStream(ctx.stream)
    jobs = []
    for seed in (1, 2):
        x = torch.from_numpy(rng.standard_normal((9, 4096)).astype(np.float32)).cuda()
        w, _ = _random_matrix(fx, rng, 500, 4096, 16)
        q = Matrix(fx, 9, 4096, 16)
        outs = [torch.zeros(9, 4096, device="cuda"), torch.zeros(9, 500, device="cuda"), torch.zeros(9, 500, device="cuda")]

        def run(x=x, w=w, q=q, outs=outs):
            ctx.fp4_quantize(x.data_ptr(), fx.F32, 4096, q.h)
            ctx.fp4_dequantize(q.h, outs[0].data_ptr(), fx.F32, 4096)
            ctx.gemm_fp4(q.h, w.h, outs[1].data_ptr(), fx.F32, 500)
            ctx.gemv_fp4(x.data_ptr(), fx.F32, 4096, 9, w.h, outs[2].data_ptr(), fx.F32, 500)

        torch.cuda.synchronize()
        run()
        ctx.sync()
        eager = [o.clone() for o in outs]
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            run()
        jobs.append((graph, outs, eager, q, x, w))
    for _ in range(3):
        for _, outs, _, _, _, _ in jobs:
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for graph, _, _, _, _, _ in jobs:
                graph.replay()
        ctx.sync()
        for _, outs, eager, _, _, _ in jobs:
            assert all(torch.equal(o, e) for o, e in zip(outs, eager))


@pytest.mark.parametrize("M,N,K", [(1, 2560, 9728), (5, 700, 20000), (64, 300, 9000), (130, 1000, 5000), (1100, 2300, 2000)])
def test_products_repeat_bit_for_bit(fx, ctx, M, N, K):
    """Split sums are added in a fixed order."""
    rng = np.random.default_rng(M + K)
    x, _ = _random_matrix(fx, rng, M, K, 16)
    w, _ = _random_matrix(fx, rng, N, K, 16)
    xs = torch.from_numpy(rng.standard_normal((min(M, 16), K)).astype(np.float32)).cuda()
    first = None
    for _ in range(4):
        a, b = torch.zeros(M, N, device="cuda"), torch.zeros(min(M, 16), N, device="cuda")
        torch.cuda.synchronize()
        ctx.gemm_fp4(x.h, w.h, a.data_ptr(), fx.F32, N)
        ctx.gemv_fp4(xs.data_ptr(), fx.F32, K, min(M, 16), w.h, b.data_ptr(), fx.F32, N)
        ctx.sync()
        assert first is None or (torch.equal(a, first[0]) and torch.equal(b, first[1]))
        first = (a, b)


@pytest.mark.parametrize("fmt", [16, 32])
def test_offsets_beyond_32_bits(fx, ctx, fmt):
    """The last rows of matrices of more than 2^32 bytes and 2^31 elements come out as they do alone."""
    rows, cols, tail, K = 300003, 8192, 259, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    x[:-tail] = 1.0
    x[-tail:] = torch.randn(tail, cols, device="cuda", generator=g).bfloat16()
    assert rows * cols > 2 ** 31
    nc, ns = fx.fp4_bytes(rows, cols, fmt)
    codes, scales = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
    q = fx.Fp4(codes.data_ptr(), scales.data_ptr(), rows, cols, fmt, 1.0)
    small = Matrix(fx, tail, cols, fmt)
    out, alone = torch.zeros_like(x), torch.zeros(tail, cols, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_quantize(x.data_ptr(), fx.BF16, cols, q)
    ctx.fp4_dequantize(q, out.data_ptr(), fx.BF16, cols)
    ctx.fp4_quantize(x[-tail:].data_ptr(), fx.BF16, cols, small.h)
    ctx.fp4_dequantize(small.h, alone.data_ptr(), fx.BF16, cols)
    ctx.sync()
    ones = ref.values(*ref.quantize(np.ones((1, fmt)), fmt), fmt)[0, 0]  # 6 * e4m3(1 / 6) for blocks of 16
    assert torch.equal(out[-tail:], alone) and (out[:-tail] == ones).all()
    # as weights: the last columns of a product, its rows past 2^32 bytes with them
    first = torch.randn(3, cols, device="cuda", generator=g).bfloat16()
    a = Matrix(fx, 3, cols, fmt)
    full, part = torch.zeros(3, rows, device="cuda"), torch.zeros(3, tail, device="cuda")
    few, few_part = torch.zeros(3, rows, device="cuda"), torch.zeros(3, tail, device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_quantize(first.data_ptr(), fx.BF16, cols, a.h)
    ctx.gemm_fp4(a.h, q, full.data_ptr(), fx.F32, rows)
    ctx.gemm_fp4(a.h, small.h, part.data_ptr(), fx.F32, tail)
    ctx.gemv_fp4(first.data_ptr(), fx.BF16, cols, 3, q, few.data_ptr(), fx.F32, rows)
    ctx.gemv_fp4(first.data_ptr(), fx.BF16, cols, 3, small.h, few_part.data_ptr(), fx.F32, tail)
    ctx.sync()
    del x
    # other splits of K: sums in another order, of 8192 products
    scale = (first.float().abs().sum(1, keepdim=True) * 8.0)
    assert ((full[:, -tail:] - part).abs() <= scale * 2.0 ** -18).all()
    assert ((few[:, -tail:] - few_part).abs() <= scale * 2.0 ** -18).all()
    # as rows, into an output of more than 2^31 elements
    xa = Matrix(fx, rows, K, fmt)
    rnd = torch.randn(rows, K, device="cuda", generator=g).bfloat16()
    wa = Matrix(fx, cols, K, fmt)
    wr = torch.randn(cols, K, device="cuda", generator=g).bfloat16()
    torch.cuda.synchronize()
    ctx.fp4_quantize(rnd.data_ptr(), fx.BF16, K, xa.h)
    ctx.fp4_quantize(wr.data_ptr(), fx.BF16, K, wa.h)
    ctx.gemm_fp4(xa.h, wa.h, out.data_ptr(), fx.BF16, cols)
    last = Matrix(fx, tail, K, fmt)
    ctx.fp4_quantize(rnd[-tail:].data_ptr(), fx.BF16, K, last.h)
    ctx.gemm_fp4(last.h, wa.h, alone.data_ptr(), fx.BF16, cols)
    ctx.sync()
    assert torch.equal(out[-tail:], alone)  # one k-slice: the same sums


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_calls_run_on_the_contexts_device(fx):
    """Whatever device is current, a context's calls run on its own, and leave the current one as it was."""
    other = fx.Context(1)
    torch.cuda.set_device(0)
    x = torch.ones(4, 64, device="cuda:1")
    codes, scales = torch.zeros(4 * 32, dtype=torch.uint8, device="cuda:1"), torch.zeros(512, dtype=torch.uint8, device="cuda:1")
    q = fx.Fp4(codes.data_ptr(), scales.data_ptr(), 4, 64, 16, 1.0)
    out = torch.zeros(4, 4, device="cuda:1")
    torch.cuda.synchronize(1)
    other.fp4_quantize(x.data_ptr(), fx.F32, 64, q)
    other.gemm_fp4(q, q, out.data_ptr(), fx.F32, 4)
    other.sync()
    assert (out == 64).all() and torch.cuda.current_device() == 0
    other.close()


def test_two_contexts_at_once(fx, ctx):
    """Products on two contexts' streams at the same time share nothing."""
    other = fx.Context(0)
    rng = np.random.default_rng(12)
    jobs = []
    for c in (ctx, other):
        x, xv = _random_matrix(fx, rng, 33, 4096, 16)
        w, wv = _random_matrix(fx, rng, 256, 4096, 16)
        jobs.append((c, x, w, xv, wv, torch.zeros(33, 256, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(20):
        for c, x, w, _, _, out in jobs:
            c.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, 256)
    for c, x, w, xv, wv, out in jobs:
        c.sync()
        want = xv @ wv.T
        assert (np.abs(out.double().cpu().numpy() - want) <= _product_tolerance(xv, wv, want, "f32", None, None)).all()
    other.close()

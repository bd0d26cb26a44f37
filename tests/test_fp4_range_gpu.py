"""The 4-bit operators where f32 ends: matrix scales at both ends of their range, values and sums that leave the normal range
on the way to a result that does not, the single rounding of values that are read back, and sums whose every bit is known."""
import numpy as np
import pytest
import torch

import fp4_reference as ref
from test_fp4_gpu import TORCH, Matrix, _dt, _plain

pytestmark = pytest.mark.gpu

F32_MAX = float(np.finfo(np.float32).max)


# ---------------------------------------------------------------------------------------------------- quantising
def _whole_range(rng, fmt, k, name):
    """Blocks whose maxima go through the whole range of the type, and next to every border of the codes for the smallest
    power-of-two factor under a scale of 2^k."""
    lo, hi = {"f32": (-149, 127), "bf16": (-133, 127), "f16": (-24, 15)}[name]
    rows = []
    for e in range(lo, hi + 1):
        r = rng.uniform(1, 2, fmt) * np.exp2(e - rng.integers(0, 7, fmt)) * rng.choice([-1, 1], fmt)
        r[rng.integers(0, fmt)] = 1.99 * 2.0 ** e if e > lo else 2.0 ** e
        rows.append(r)
    if name == "f32":
        for border in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0):
            t = border * 2.0 ** (k - 127)
            if 2.0 ** -126 <= t < 2.0 ** 120:
                t = np.float32(t)
                r = np.zeros(fmt)
                r[:3] = np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(1))
                rows.append(r)
    if name != "f16":
        rows.append(np.full(fmt, 1e30))
        rows.append(np.where(np.arange(fmt) == 3, -3.3e38 if name == "f32" else -3e38, 1.0))
    rows.append(np.where(np.arange(fmt) == 1, np.inf, 1.0))
    rows.append(np.where(np.arange(fmt) == 2, np.nan, 1.0))
    return np.array(rows)


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("k", [-100, -40, -23, -2, -1, 1, 2, 23, 40, 100])
def test_quantize_with_every_size_of_scale(fx, ctx, k, name, fmt):
    """x / scale is exact, whatever f32 makes of it: a quotient beyond the f32 range is a large value like any other (the
    largest factor, codes of 6), and one below the normal range is rounded once, by the code. Only x that is not finite
    makes a block NaN."""
    dev, x = _plain(_whole_range(np.random.default_rng(k + 1000), fmt, k, name), name, fmt)
    q = Matrix(fx, x.shape[0], fmt, fmt, 2.0 ** k)
    torch.cuda.synchronize()
    ctx.fp4_quantize(dev.data_ptr(), _dt(fx, name), fmt, q.h)
    ctx.sync()
    code, byte, clean = q.read()
    want, wbyte = ref.quantize(x, fmt, 2.0 ** k)
    assert clean
    assert (byte == wbyte).all()
    assert np.array_equal(ref.values(code, byte, fmt), ref.values(want, wbyte, fmt), equal_nan=True)


# ---------------------------------------------------------------------------------------------------- products
def _exact_matrix(fx, rng, rows, cols, fmt, e, scale):
    """Codes of 0, +-0.5 .. +-6 under one power-of-two factor 2^e: any sum of a few thousand products of two of them is an
    exact f32 number. The last row is 0. -> the matrix and its values without the scale."""
    code = rng.integers(0, 16, (rows, cols))
    code[-1] = 0
    nb = -(-cols // fmt)
    b = (e + 127) if fmt == 32 else (e + 7) << 3
    byte = np.full((rows, nb), b, np.uint8)
    return Matrix(fx, rows, cols, fmt, scale, ref.pack(code, byte)), ref.values(code, byte, fmt)


def _f32(v):
    """float64 -> the nearest f32, infinity beyond it."""
    with np.errstate(over="ignore"):
        return v.astype(np.float32).astype(np.float64)


SHAPES = [(5, 130, 600), (1, 40, 64), (24, 260, 6000), (130, 300, 3000), (1300, 2200, 300)]  # alone, split, in pairs of CTAs


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("fmt,ex,ew,sx,sw", [
    (16, 0, 0, 2.0 ** 70, 2.0 ** 70),               # beyond f32, but for the rows and columns of zeros
    (16, -6, -6, 2.0 ** 60, 2.0 ** 70),             # only the scales' product is
    (32, -60, -60, 2.0 ** 100, 2.0 ** 100),
    (32, -60, -60, -2.0 ** 127, 2.0 ** 65),
    (32, 40, 40, 2.0 ** -100, 2.0 ** -60),          # only the scales' product is below it
    (32, 50, 50, 2.0 ** -100, 2.0 ** -100),
    (32, 50, 50, 2.0 ** -149, 2.0 ** -40),
    (32, 20, 20, 1.7 * 2.0 ** -140, 1.3 * 2.0 ** 5),  # neither is, but the product has few digits left
    (32, 0, 20, 2.0 ** 100, 1.9 * 2.0 ** -149),
    (16, 3, 3, 2.0 ** -100, 2.0 ** -100),           # nothing is left
    (16, 2, -2, 0.75, 1.7), (32, 100, -100, 2.0 ** 30, 2.0 ** -31), (16, 0, 0, 0.0, 2.0 ** 100)])
def test_product_with_every_size_of_scale(fx, ctx, fmt, ex, ew, sx, sw, M, N, K):
    """The sum times the two scales, whatever f32 makes of the scales' own product. The sums are exact; then at most three
    roundings of 2^-24, and half of the smallest step where the result is subnormal."""
    rng = np.random.default_rng(M + N + K)
    x, xv = _exact_matrix(fx, rng, M, K, fmt, ex, sx)
    w, wv = _exact_matrix(fx, rng, N, K, fmt, ew, sw)
    out = torch.full((M + 1, N), 7.0, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, N)
    ctx.sync()
    want = (xv @ wv.T) * (float(np.float32(sx)) * float(np.float32(sw)))
    got = out[:M].double().cpu().numpy()
    assert (out[M:] == 7).all()
    beyond = np.isinf(_f32(want))
    assert (got[beyond] == np.sign(want[beyond]) * np.inf).all()
    fine = ~beyond
    assert (np.abs(got - want)[fine] <= 3 * 2.0 ** -24 * np.abs(want)[fine] + 2.0 ** -149).all()


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("fmt,ex,ew,sx,sw,eg", [
    (32, 40, 40, 2.0 ** -50, 2.0 ** -50, -35),   # scales * gate has few digits left
    (32, 40, 40, 2.0 ** -60, 2.0 ** -60, -100),  # or none
    (32, -50, -50, 2.0 ** 50, 2.0 ** 50, 40),    # or is beyond f32
    (32, -60, -60, 2.0 ** 100, 2.0 ** 100, -70),
    (32, 50, 50, 2.0 ** -100, 2.0 ** -100, 70),
    (16, 0, 0, 2.0 ** 60, 2.0 ** 60, -60),        # the scales alone take the sum out of f32
    (16, 0, 0, 2.0 ** 90, 1.3 * 2.0 ** 90, -149 + 23),
    (32, 50, 50, 2.0 ** -127, 2.0 ** -127, 100),
    (32, 50, 50, 1.7 * 2.0 ** -140, 2.0 ** -120, 120),
    (32, -60, -60, 2.0 ** 120, 2.0 ** 120, -30),
    (16, 0, 0, 0.5, 1.7, 0)])
def test_gated_product_with_every_size_of_scale(fx, ctx, fmt, ex, ew, sx, sw, eg, in_place, M, N, K):
    """gate and residual: one rounding more, and that of the sum with the residual. A gate of 0 leaves the residual."""
    rng = np.random.default_rng(M + N + K + 1)
    x, xv = _exact_matrix(fx, rng, M, K, fmt, ex, sx)
    w, wv = _exact_matrix(fx, rng, N, K, fmt, ew, sw)
    gate = (rng.uniform(1, 2, N) * rng.choice([-1, 1], N) * 2.0 ** eg).astype(np.float32)
    gate[::7] = 0
    term = gate.astype(np.float64) * ((xv @ wv.T) * (float(np.float32(sx)) * float(np.float32(sw))))
    residual = (rng.standard_normal((M, N)) * np.abs(term).mean()).astype(np.float32)
    want = residual.astype(np.float64) + term
    g, r = torch.from_numpy(gate).cuda(), torch.from_numpy(residual).cuda()
    out = r.clone() if in_place else torch.zeros(M, N, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, N, gate_ptr=g.data_ptr(),
                 residual_ptr=out.data_ptr() if in_place else r.data_ptr(), ld_residual=N)
    ctx.sync()
    got = out.double().cpu().numpy()
    assert (np.abs(got - want) <= 4 * 2.0 ** -24 * np.abs(term) + 2.0 ** -24 * np.abs(want) + 2.0 ** -149).all()
    assert (got[:, ::7] == residual[:, ::7]).all()


# ---------------------------------------------------------------------------------------------------- few rows
@pytest.mark.parametrize("xname", ["f32", "bf16"])
@pytest.mark.parametrize("fmt,e,ex,scale", [
    (16, 7, 120, 2.0 ** -60), (16, 7, 120, 2.0 ** -100), (16, -6, -100, 2.0 ** 125), (16, 0, -100, 2.0 ** 127),
    (32, 7, 100, 2.0 ** -60), (32, -20, -80, 2.0 ** 127), (32, 100, -90, 2.0 ** -100), (16, 0, 100, 2.0 ** -149)])
def test_few_row_product_with_every_size_of_scale(fx, ctx, fmt, e, ex, scale, xname):
    """The matrix's scale comes to the sum in one step: sums that it brings back into the f32 range are not lost before.
    x of one code's step and codes under one factor: exact sums and, by a power of two, exact results."""
    rng = np.random.default_rng(7)
    w, wv = _exact_matrix(fx, rng, 70, 200, fmt, e, scale)
    dev, x = _plain(rng.integers(-3, 4, (5, 200)) * 2.0 ** ex, xname, 200)
    out = torch.zeros(5, 70, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), _dt(fx, xname), 200, 5, w.h, out.data_ptr(), fx.F32, 70)
    ctx.sync()
    want = (x @ wv.T) * scale
    assert np.isfinite(_f32(want)).all()
    assert (np.abs(out.double().cpu().numpy() - want) <= 2.0 ** -149).all()


@pytest.mark.parametrize("fmt,e", [(32, 100), (32, 125), (32, 0), (16, 7)])
@pytest.mark.parametrize("ex", [-149, -140, -130, -126, -122, -118, -110, -100])
def test_few_row_product_of_tiny_rows(fx, ctx, ex, fmt, e):
    """f32 x down to the smallest subnormal numbers keeps its digits where the weights make something of it, but for the digit
    2^-149. Sums as in test_fp4_gpu._few_row_tolerance for 64 columns, with steps of 2^-149 (blocks of 16, whose sums are held
    times 2^-16: 2^-133) per product below the normal range."""
    rng = np.random.default_rng(ex + 500)
    K = 64
    w, wv = _exact_matrix(fx, rng, 40, K, fmt, e, 1.0)
    dev, x = _plain(rng.uniform(1, 2, (4, K)) * rng.choice([-1, 1], (4, K)) * 2.0 ** ex, "f32", K)
    out = torch.zeros(4, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), fx.F32, K, 4, w.h, out.data_ptr(), fx.F32, 40)
    ctx.sync()
    want = x @ wv.T
    mag = np.abs(x) @ np.abs(wv).T
    tol = mag * (2 * 3 * 4 + 8) * 2.0 ** -23 + 2.0 ** -149 * np.abs(wv).sum(1) + 3 * K * (2.0 ** -133 if fmt == 16 else 2.0 ** -149)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


# ---------------------------------------------------------------------------------------------------- reading back
def _round_once(v, name):
    """float64 -> the nearest value of a type, ties to even, as float64; f16 saturates."""
    p, low, top = {"f32": (24, -126, F32_MAX), "f16": (11, -14, 65504.0),
                   "bf16": (8, -126, float(torch.finfo(torch.bfloat16).max))}[name]
    e = np.maximum(np.frexp(v)[1] - 1, low).astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        step = np.exp2(e - (p - 1))
        r = np.round(v / step) * step
    return np.where(np.abs(r) > top, np.copysign(65504.0 if name == "f16" else np.inf, v), r)


def _scales_next_to_ties():
    """f32 scales whose product with 3 lies next to the middle of two neighbours of a 16-bit type, nearer than an f32 can
    tell: 3 s = t +- 1/4 unit of f32, t such a middle."""
    out = []
    for bits in (8, 11):
        cut = 24 - bits
        for top in range(2 ** (bits - 1), 2 ** bits, 2 ** (bits - 1) // 64):
            for odd, d in ((0, 1), (1, -1)):  # a tie would go to the even neighbour; this does not
                t = (((top | 1) - 1 + odd) << cut | 1 << (cut - 1)) * 4 + d
                if t % 3 == 0:
                    out.append(t // 3 * 2.0 ** -24)
    return [s for s in out if float(np.float32(s)) == s]


def _read_back(fx, ctx, m, rows, cols, name, pad):
    out = torch.zeros(rows, cols + pad, dtype=TORCH[name], device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_dequantize(m.h, out.data_ptr(), _dt(fx, name), cols + pad)
    ctx.sync()
    return out[:, :cols].double().cpu().numpy()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -60, 2.0 ** 90, 0.3, -1.7, 1.1 * 2.0 ** -100, 1.9 * 2.0 ** -120, 1.3 * 2.0 ** 100,
                                   F32_MAX, 2.0 ** -126, 3 * 2.0 ** -149, 2.0 ** -149, 1.234 * 2.0 ** -135, 0.0])
def test_dequantize_rounds_once(fx, ctx, scale, name, fmt):
    """Every code with every factor and a matrix scale from anywhere in the f32 range: the nearest value of the type, also
    among the subnormal ones."""
    code = np.tile(np.arange(16), (256, fmt // 16 * 3))
    byte = np.repeat(np.arange(256)[:, None], 3, 1).astype(np.uint8)
    if fmt == 16:
        byte &= 127
    m = Matrix(fx, 256, code.shape[1], fmt, scale, ref.pack(code, byte))
    want = _round_once(ref.values(code, byte, fmt, float(np.float32(scale))), name)
    for pad in (0, 1):
        got = _read_back(fx, ctx, m, 256, code.shape[1], name, pad)
        assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_dequantize_next_to_ties(fx, ctx, name, fmt):
    scales = _scales_next_to_ties()
    assert len(scales) >= 40
    code = np.tile(np.arange(16), (4, 4))
    byte = np.tile(np.array([127, 128, 120, 126] if fmt == 32 else [0x38, 0x30, 0x3C, 0x48])[:, None], (1, 64 // fmt)).astype(np.uint8)
    for s in scales:
        m = Matrix(fx, 4, 64, fmt, s, ref.pack(code, byte))
        want = _round_once(ref.values(code, byte, fmt, s), name)
        assert (_read_back(fx, ctx, m, 4, 64, name, 0) == want).all()


# ---------------------------------------------------------------------------------------------------- the largest sizes
@pytest.mark.parametrize("fmt", [16, 32])
def test_rows_as_long_as_an_int_allows(fx, ctx, fmt):
    """One row of 2^31 - 7 columns: rounding that up to tiles takes more than 31 bits. Its last columns come out as they do
    alone."""
    cols, start = 2 ** 31 - 7, 2 ** 31 - 1024
    x = torch.ones(1, cols, dtype=torch.bfloat16, device="cuda")
    x[0, start:] = torch.randn(cols - start, device="cuda").bfloat16()
    nc, ns = fx.fp4_bytes(1, cols, fmt)
    codes, scales = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
    q = fx.Fp4(codes.data_ptr(), scales.data_ptr(), 1, cols, fmt, 1.0)
    tail = Matrix(fx, 1, cols - start, fmt)
    alone = torch.zeros(1, cols - start, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ctx.fp4_quantize(x.data_ptr(), fx.BF16, cols, q)
    ctx.fp4_quantize(x[:, start:].data_ptr(), fx.BF16, cols - start, tail.h)
    ctx.fp4_dequantize(tail.h, alone.data_ptr(), fx.BF16, cols - start)
    ctx.sync()
    assert torch.equal(codes[start // 2:], tail.codes[:tail.nc])
    x.zero_()
    torch.cuda.synchronize()
    ctx.fp4_dequantize(q, x.data_ptr(), fx.BF16, cols)
    ctx.sync()
    one = ref.values(*ref.quantize(np.ones((1, fmt)), fmt), fmt)[0, 0]
    assert torch.equal(x[:, start:], alone) and (x[:, :start] == one).all()
    del x, codes, scales
    torch.cuda.empty_cache()


def test_as_many_rows_as_an_int_allows(fx, ctx):
    """A product of 2^31 - 7 rows, every one of them right."""
    rows = 2 ** 31 - 7
    nc, ns = fx.fp4_bytes(rows, 32, 16)
    codes = torch.full((nc,), 0x22, dtype=torch.uint8, device="cuda")  # 1
    codes[-300 * 16:] = 0x44                                           # 2
    scales = torch.full((ns // 4,), 0x3838, dtype=torch.int32, device="cuda")  # two blocks of factor 1, then padding
    scales[-128:].view(32, 4)[32 - 7:, 3] = 0  # the rows past the end
    x = fx.Fp4(codes.data_ptr(), scales.data_ptr(), rows, 32, 16, 1.0)
    w = Matrix(fx, 1, 32, 16, 1.0, ref.pack(np.full((1, 32), 2), np.full((1, 2), 0x38, np.uint8)))
    out = torch.zeros(rows, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x, w.h, out.data_ptr(), fx.F16, 1)
    ctx.sync()
    assert (out[:-300] == 32).all() and (out[-300:] == 64).all()
    del codes, scales, out
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------------- errors
def test_an_earlier_error_of_the_thread_is_not_a_failed_launch(fx, ctx):
    """A refused runtime call of the program's own (here: a device that does not exist) leaves an error that the next reader
    gets. The operators' launches answer for themselves."""
    import ctypes
    runtime = ctypes.CDLL("libcudart.so.12")
    x = torch.ones(4, 64, device="cuda")
    q, out = Matrix(fx, 4, 64, 16), torch.zeros(4, 64, device="cuda")
    torch.cuda.synchronize()
    try:
        for call in (lambda: ctx.fp4_quantize(x.data_ptr(), fx.F32, 64, q.h),
                     lambda: ctx.fp4_dequantize(q.h, out.data_ptr(), fx.F32, 64),
                     lambda: ctx.gemm_fp4(q.h, q.h, out.data_ptr(), fx.F32, 64),
                     lambda: ctx.gemv_fp4(x.data_ptr(), fx.F32, 64, 4, q.h, out.data_ptr(), fx.F32, 64)):
            assert runtime.cudaSetDevice(10 ** 6) != 0
            call()
            assert runtime.cudaGetLastError() != 0  # and it is still there for its own reader
    finally:
        runtime.cudaGetLastError()
    ctx.sync()


def test_a_failed_launch_names_its_cause(fx, ctx):
    """Launches into a capture that the program has spoilt (by waiting for the stream inside of it) are refused by the runtime,
    and the refusal's own text comes back; afterwards everything works as before."""
    import ctypes
    runtime = ctypes.CDLL("libcudart.so.12")
    runtime.cudaGetErrorString.restype = ctypes.c_char_p
    x = torch.ones(4, 64, device="cuda")
    q, out = Matrix(fx, 4, 64, 16), torch.zeros(4, 64, device="cuda")
    few = torch.zeros(4, 4, device="cuda")
    calls = (lambda: ctx.fp4_quantize(x.data_ptr(), fx.F32, 64, q.h),
             lambda: ctx.fp4_dequantize(q.h, out.data_ptr(), fx.F32, 64),
             lambda: ctx.gemm_fp4(q.h, q.h, few.data_ptr(), fx.F32, 4),
             lambda: ctx.gemv_fp4(x.data_ptr(), fx.F32, 64, 4, q.h, few.data_ptr(), fx.F32, 4))
    torch.cuda.synchronize()
    for call in calls:
        stream, graph = ctypes.c_void_p(ctx.stream), ctypes.c_void_p()
        assert runtime.cudaStreamBeginCapture(stream, 2) == 0
        spoilt = runtime.cudaStreamSynchronize(stream)
        runtime.cudaGetLastError()
        try:
            with pytest.raises(fx.FluxCudaError) as e:
                call()
        finally:
            runtime.cudaStreamEndCapture(stream, ctypes.byref(graph))
            runtime.cudaGetLastError()
        assert spoilt != 0
        assert "launch failed" in str(e.value) and runtime.cudaGetErrorString(901).decode() in str(e.value)
    for call in calls:
        call()
    ctx.sync()
    assert (few == 64 * ref.values(*ref.quantize(np.ones((1, 64)), 16), 16)[0, 0]).all()  # ones are 6 * e4m3(1 / 6)


# ---------------------------------------------------------------------------------------------------- sums known to the bit
def _sparse(rng, rows, cols, fmt):
    """Codes +-1 with factor 1 and a value per row and column: a lost or doubled column changes every sum."""
    code = rng.choice([2, 10], (rows, cols))
    byte = np.full((rows, -(-cols // fmt)), 127 if fmt == 32 else 0x38, np.uint8)
    return code, byte


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("xname", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 60000), (3, 20000), (16, 30000), (1, 65536), (5, 65536), (7, 9216), (16, 9216), (2, 65505)])
def test_few_row_product_of_long_rows_to_the_bit(fx, ctx, M, K, xname, fmt):
    """Whole numbers of at most 7 bits times +-1: every partial sum is an exact f32 number (below 2^24), so the result is
    exact however the sum is split, and no column may be lost or counted twice."""
    rng = np.random.default_rng(K + M)
    code, byte = _sparse(rng, 40, K, fmt)
    w, wv = Matrix(fx, 40, K, fmt, 1.0, ref.pack(code, byte)), ref.values(code, byte, fmt)
    dev, x = _plain(rng.integers(1, 128, (M, K)).astype(np.float64), xname, K)
    out = torch.zeros(M, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), _dt(fx, xname), K, M, w.h, out.data_ptr(), fx.F32, 40)
    ctx.sync()
    assert (out.double().cpu().numpy() == x @ wv.T).all()


@pytest.mark.parametrize("M,K", [(1, 60000), (3, 20000), (1, 65536), (5, 65536), (4, 9216)])
def test_few_row_product_adds_short_chains(fx, ctx, M, K):
    """The tensor instruction may truncate, the additions of its chains round. All numbers are positive, so that truncation
    adds up and no cancellation widens the bound. A chain is 128 columns, 8 instructions for each part of x, an instruction
    truncates what it has added up and its aligned products: 2 * 2^-23 of the chain each. The chains and the pieces of a
    sum (40 at most: 16 warps twice, 8 CTAs) are added with n = K / 128 + 40 roundings of at most 2^-24 of the sum either way;
    6 sqrt(n) of those are exceeded once in 10^7 (Hoeffding)."""
    rng = np.random.default_rng(K)
    code, byte = ref.quantize(np.abs(rng.standard_normal((40, K))), 16)
    w, wv = Matrix(fx, 40, K, 16, 1.0, ref.pack(code, byte)), ref.values(code, byte, 16)
    dev, x = _plain(np.abs(rng.standard_normal((M, K))), "f32", K)
    out = torch.zeros(M, 40, device="cuda")
    torch.cuda.synchronize()
    ctx.gemv_fp4(dev.data_ptr(), fx.F32, K, M, w.h, out.data_ptr(), fx.F32, 40)
    ctx.sync()
    want = x @ wv.T
    tol = want * (8 * 2 * 2.0 ** -23 + 6 * np.sqrt(K / 128 + 40) * 2.0 ** -24)
    assert (np.abs(out.double().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("M,N,K", [(1, 130, 60000), (20, 200, 9000), (40, 140, 20001), (100, 260, 9216), (130, 300, 5000),
                                   (300, 500, 9999), (1025, 2049, 1600), (1300, 2200, 300), (16, 20000, 600), (2600, 5200, 64)])
def test_product_to_the_bit(fx, ctx, M, N, K, fmt):
    """Codes under factors 1 and 2: sums of at most 2^24 quarters are exact f32 numbers, so the result is exact however the sum is
    split, and every block needs its own factor."""
    rng = np.random.default_rng(M + N + K)

    def matrix(rows):
        code = rng.choice([0, 1, 2, 9, 10, 3, 11], (rows, K))  # 0, +-0.5, +-1, +-1.5
        byte = rng.choice([127, 128] if fmt == 32 else [0x38, 0x40], (rows, -(-K // fmt))).astype(np.uint8)
        return Matrix(fx, rows, K, fmt, 1.0, ref.pack(code, byte)), ref.values(code, byte, fmt)

    x, xv = matrix(M)
    w, wv = matrix(N)
    assert (np.abs(xv).sum(1) * 3).max() < 2 ** 22
    out = torch.zeros(M, N, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, N)
    ctx.sync()
    want = (torch.from_numpy(xv).cuda() @ torch.from_numpy(wv).cuda().T).cpu().numpy()
    assert (out.double().cpu().numpy() == want).all()


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("side", ["w", "x"])
@pytest.mark.parametrize("M,K", [(16, 32), (128, 32), (200, 300)])
def test_product_with_every_factor(fx, ctx, M, K, side, fmt):
    """Every finite factor with every code on the tensor cores, against rows that pick out one column each: single exact products.
    Results below the normal range may be lost (2^-126 in all); what lies beyond the f32 range is left out; NaN stays in its row."""
    code = np.tile(np.arange(16), (256, -(-K // 16)))[:, :K]
    byte = np.repeat(np.arange(256)[:, None], -(-K // fmt), 1).astype(np.uint8)
    if fmt == 16:
        byte &= 127
    every, ev = Matrix(fx, 256, K, fmt, 1.0, ref.pack(code, byte)), ref.values(code, byte, fmt)
    at = np.arange(M) * 7 % K
    pcode = np.zeros((M, K), np.int64)
    pcode[np.arange(M), at] = 2
    pbyte = np.full((M, -(-K // fmt)), 127 if fmt == 32 else 0x38, np.uint8)
    pick = Matrix(fx, M, K, fmt, 1.0, ref.pack(pcode, pbyte))
    out = torch.zeros((M, 256) if side == "w" else (256, M), device="cuda")
    torch.cuda.synchronize()
    if side == "w":
        ctx.gemm_fp4(pick.h, every.h, out.data_ptr(), fx.F32, 256)
    else:
        ctx.gemm_fp4(every.h, pick.h, out.data_ptr(), fx.F32, M)
    ctx.sync()
    got = out.double().cpu().numpy()
    got = got if side == "w" else got.T
    want = ev[:, at].T
    inside = np.isnan(ev).any(1) | (np.abs(ev).max(1) < F32_MAX)
    assert inside.sum() >= 252
    assert (np.isnan(got) == np.isnan(want))[:, inside].all()
    fine = np.broadcast_to(inside, want.shape) & np.isfinite(want)
    small = fine & (np.abs(want) < 2.0 ** -126)
    assert (got == want)[fine & ~small].all()
    assert (np.abs(got - want)[small] <= 2.0 ** -126).all()


@pytest.mark.parametrize("e", [-125, -100, -60, -1, 0, 1, 60, 100, 125])
def test_product_of_opposite_factors(fx, ctx, e):
    """2^e against 2^-e: products near 1, however far the factors are from it."""
    rng = np.random.default_rng(e + 200)
    x, xv = _exact_matrix(fx, rng, 20, 512, 32, e, 1.0)
    w, wv = _exact_matrix(fx, rng, 140, 512, 32, -e, 1.0)
    out = torch.zeros(20, 140, device="cuda")
    torch.cuda.synchronize()
    ctx.gemm_fp4(x.h, w.h, out.data_ptr(), fx.F32, 140)
    ctx.sync()
    assert (out.double().cpu().numpy() == xv @ wv.T).all()


# ---------------------------------------------------------------------------------------------------- five rows and more
def _weights_of_ones(fx, N, K, fmt):
    """+-1 with factors 1 and 2, made on the device, and its values in 64 bits."""
    g = torch.Generator(device="cuda").manual_seed(N + K)
    sign = torch.randint(0, 2, (N, K), device="cuda", generator=g, dtype=torch.uint8)
    code = torch.zeros(N, 32 * -(-K // 32), dtype=torch.uint8, device="cuda")
    code[:, :K] = 2 | sign << 3
    up = torch.randint(0, 2, (N, -(-K // fmt)), device="cuda", generator=g, dtype=torch.uint8)
    m = Matrix(fx, N, K, fmt)
    m.codes[:m.nc] = (code[:, 0::2] | code[:, 1::2] << 4).reshape(-1)
    byte = (127 + up) if fmt == 32 else (0x38 + 8 * up)
    tiles, chunks = -(-N // 128), -(-up.shape[1] // 4)
    full = torch.zeros(tiles * 128, chunks * 4, dtype=torch.uint8, device="cuda")
    full[:N, :up.shape[1]] = byte
    m.scales[:m.ns] = full.view(tiles, 4, 32, chunks, 4).permute(0, 3, 2, 1, 4).reshape(-1)
    values = (1.0 - 2.0 * sign.double()) * (1.0 + up.double()).repeat_interleave(fmt, 1)[:, :K]
    return m, values


@pytest.mark.parametrize("fmt", [16, 32])
@pytest.mark.parametrize("N,K", [(18432, 9216), (19456, 2560), (2560, 9728), (5000, 4001)])
def test_few_row_product_of_every_number_of_rows(fx, ctx, N, K, fmt):
    """Every number of rows and type, so every way to lay them out: sets of rows, splits of K, several rounds of clusters. Whole
    numbers of a sum of magnitudes below 2^24: exact."""
    w, wv = _weights_of_ones(fx, N, K, fmt)
    g = torch.Generator(device="cuda").manual_seed(7)
    for name in ("bf16", "f16", "f32"):
        for m in range(1, 17):
            x = torch.randint(-127, 128, (m, K), device="cuda", generator=g).to(TORCH[name])
            out = torch.full((m + 1, N), 7.0, device="cuda")
            torch.cuda.synchronize()
            ctx.gemv_fp4(x.data_ptr(), _dt(fx, name), K, m, w.h, out.data_ptr(), fx.F32, N)
            ctx.sync()
            assert (out[:m].double() == x.double() @ wv.T).all() and (out[m:] == 7).all(), (name, m)


@pytest.mark.parametrize("N,K", [(18432, 9216), (19456, 2560), (9728, 2560), (2560, 9728)])
def test_more_rows_cost_no_more_than_calls_of_four(fx, ctx, N, K):
    """One call of 5 to 16 rows is not slower than as many calls of four rows as they make (a quarter is allowed for noise).
    Weights of more than the caches hold are gone through in turn."""
    sets = max(2, int(3e8 / (0.56 * N * K)))
    ws = [Matrix(fx, N, K, 16) for _ in range(sets)]
    for w in ws:
        w.codes[:w.nc] = 0x22
        w.scales[:w.ns] = 0x38
    x = torch.ones(16, K, device="cuda")
    out = torch.zeros(16, N, device="cuda")
    stream = torch.cuda.ExternalStream(ctx.stream)

    def time(name, m):
        xt = x.to(TORCH[name])
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for w in ws:
                ctx.gemv_fp4(xt.data_ptr(), _dt(fx, name), K, m, w.h, out.data_ptr(), fx.F32, N)
        e = [torch.cuda.Event(enable_timing=True) for _ in range(8)]
        with torch.cuda.stream(stream):
            for ev in e:
                graph.replay()
                ev.record(stream)
        torch.cuda.synchronize()
        return min(a.elapsed_time(b) for a, b in zip(e, e[1:]))

    for name in ("bf16", "f16", "f32"):
        four = time(name, 4)
        for m in range(5, 17):
            assert time(name, m) <= 1.25 * -(-m // 4) * four, (name, m)

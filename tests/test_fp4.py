"""4-bit matrices without a GPU: buffer sizes, the refusals (the context is looked at last, so every other check answers
without one), and the test reference itself."""
import ctypes

import numpy as np
import pytest

import fp4_reference as ref

GOOD = ctypes.c_void_p(4096)  # an aligned address that is never read: the context is null


def _refused(fx, rc, text):
    assert rc == -1
    assert text in fx.lib().flux_cuda_last_error().decode()


@pytest.mark.parametrize("rows,cols,fmt,code,scale", [
    (0, 1, 16, 0, 0), (1, 1, 16, 16, 512), (1, 32, 32, 16, 512), (3, 33, 16, 96, 512), (128, 64, 16, 4096, 512),
    (129, 65, 16, 129 * 48, 2 * 2 * 512), (129, 128, 32, 129 * 64, 2 * 512), (1000, 129, 32, 1000 * 80, 8 * 2 * 512),
    (2 ** 31 - 1, 2 ** 31 - 1, 16, (2 ** 31 - 1) * 2 ** 30, 2 ** 24 * 2 ** 25 * 512)])
def test_buffer_sizes(fx, rows, cols, fmt, code, scale):
    assert fx.fp4_bytes(rows, cols, fmt) == (code, scale)


@pytest.mark.parametrize("rows,cols,fmt", [(-1, 4, 16), (4, 0, 16), (4, 4, 8), (4, 4, 0)])
def test_buffer_sizes_refuse(fx, rows, cols, fmt):
    assert fx.lib().flux_cuda_fp4_scale_bytes(rows, cols, fmt) == -1
    with pytest.raises(fx.FluxCudaError):
        fx.fp4_bytes(rows, cols, fmt)


def _matrix(fx, rows=4, cols=64, fmt=16, scale=1.0, codes=4096, scales=4096):
    return fx.Fp4(codes, scales, rows, cols, fmt, scale)


BAD = [(dict(fmt=8), "unknown format"), (dict(rows=-1), "rows >= 0"), (dict(cols=0), "cols >= 1"),
       (dict(codes=None), "no memory"), (dict(scales=None), "no memory"), (dict(codes=4104), "16-byte"),
       (dict(scales=4100), "16-byte"), (dict(scale=float("nan")), "not finite"), (dict(scale=float("inf")), "not finite")]


@pytest.mark.parametrize("change,text", BAD)
def test_bad_matrices_are_refused_everywhere(fx, change, text):
    L, bad, good = fx.lib(), _matrix(fx, **change), _matrix(fx)
    _refused(fx, L.flux_cuda_fp4_quantize(None, GOOD, 0, 64, bad), text)
    _refused(fx, L.flux_cuda_fp4_dequantize(None, bad, GOOD, 0, 64), text)
    _refused(fx, L.flux_cuda_gemm_fp4(None, bad, good, GOOD, 0, 64, None, None, 0), text)
    _refused(fx, L.flux_cuda_gemm_fp4(None, good, bad, GOOD, 0, 64, None, None, 0), text)
    _refused(fx, L.flux_cuda_gemv_fp4(None, GOOD, 0, 64, 1, bad, GOOD, 0, 64), text)


def test_null_matrices_are_refused(fx):
    L, good = fx.lib(), _matrix(fx)
    _refused(fx, L.flux_cuda_fp4_quantize(None, GOOD, 0, 64, None), "is null")
    _refused(fx, L.flux_cuda_fp4_dequantize(None, None, GOOD, 0, 64), "is null")
    _refused(fx, L.flux_cuda_gemm_fp4(None, None, good, GOOD, 0, 64, None, None, 0), "is null")
    _refused(fx, L.flux_cuda_gemm_fp4(None, good, None, GOOD, 0, 64, None, None, 0), "is null")
    _refused(fx, L.flux_cuda_gemv_fp4(None, GOOD, 0, 64, 1, None, GOOD, 0, 64), "is null")


@pytest.mark.parametrize("ptr,dtype,ld,text", [(None, 0, 64, "is null"), (4096, 3, 64, "unknown type"),
                                               (4096, -1, 64, "unknown type"), (4098, 0, 64, "not aligned"),
                                               (4097, 1, 64, "not aligned"), (4096, 0, 63, "row pitch")])
def test_bad_plain_matrices_are_refused(fx, ptr, dtype, ld, text):
    L, q = fx.lib(), _matrix(fx)
    w = _matrix(fx, rows=64)
    _refused(fx, L.flux_cuda_fp4_quantize(None, ptr, dtype, ld, q), text)
    _refused(fx, L.flux_cuda_fp4_dequantize(None, q, ptr, dtype, ld), text)
    _refused(fx, L.flux_cuda_gemm_fp4(None, q, w, ptr, dtype, ld, None, None, 0), text)
    _refused(fx, L.flux_cuda_gemv_fp4(None, ptr, dtype, ld, 2, w, GOOD, 0, 64), text)
    _refused(fx, L.flux_cuda_gemv_fp4(None, GOOD, 0, 64, 2, w, ptr, dtype, ld), text)


@pytest.mark.parametrize("scale", [0.0, 3.0, -1.0, 2.0 ** 101, 2.0 ** -101, 1.0000001])
def test_quantize_wants_a_power_of_two(fx, scale):
    _refused(fx, fx.lib().flux_cuda_fp4_quantize(None, GOOD, 0, 64, _matrix(fx, scale=scale)), "power of two")


def test_matrices_beyond_a_launch_are_refused(fx):
    L, q = fx.lib(), _matrix(fx, rows=2 ** 31 - 1, cols=2 ** 20)
    _refused(fx, L.flux_cuda_fp4_quantize(None, GOOD, 0, 2 ** 20, q), "too large")
    _refused(fx, L.flux_cuda_fp4_dequantize(None, q, GOOD, 0, 2 ** 20), "too large")


def test_product_refusals(fx):
    L = fx.lib()
    x, w = _matrix(fx), _matrix(fx, rows=8)
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, _matrix(fx, fmt=32), GOOD, 0, 64, None, None, 0), "different formats")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, _matrix(fx, cols=65), GOOD, 0, 64, None, None, 0), "different widths")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, ctypes.c_void_p(4098), None, 0), "gate is not aligned")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, None, ctypes.c_void_p(4097), 8), "residual is not aligned")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, None, GOOD, 7), "row pitch")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 1, 8, None, GOOD, 8), "residual may be out itself")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, None, GOOD, 9), "residual may be out itself")
    big = _matrix(fx, rows=2 ** 29)
    _refused(fx, L.flux_cuda_gemm_fp4(None, big, big, GOOD, 0, 2 ** 29, None, None, 0), "too many")


@pytest.mark.parametrize("rows", [-1, 17, 1000])
def test_few_row_product_takes_few_rows(fx, rows):
    _refused(fx, fx.lib().flux_cuda_gemv_fp4(None, GOOD, 0, 64, rows, _matrix(fx), GOOD, 0, 64), "0 to 16 rows")


def test_few_row_product_takes_rows_of_a_length(fx):
    w = _matrix(fx, cols=65537)
    _refused(fx, fx.lib().flux_cuda_gemv_fp4(None, GOOD, 0, 65537, 1, w, GOOD, 0, 64), "65536 columns")


def test_product_pitches(fx):
    L, x, w = fx.lib(), _matrix(fx), _matrix(fx, rows=8)
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 2 ** 30, None, None, 0), "row pitch")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, None, ctypes.c_void_p(8192), 2 ** 30), "row pitch")


def test_a_null_context_is_refused_last(fx):
    L, x, w = fx.lib(), _matrix(fx), _matrix(fx, rows=8)
    _refused(fx, L.flux_cuda_fp4_quantize(None, GOOD, 0, 64, x), "null context")
    _refused(fx, L.flux_cuda_fp4_dequantize(None, x, GOOD, 0, 64), "null context")
    _refused(fx, L.flux_cuda_gemm_fp4(None, x, w, GOOD, 0, 8, GOOD, None, 0), "null context")
    _refused(fx, L.flux_cuda_gemv_fp4(None, GOOD, 0, 64, 16, w, GOOD, 0, 8), "null context")


def test_reference_round_trip():
    """The test reference: packing is undone by unpacking, and what it quantises is within half a step of the input."""
    rng = np.random.default_rng(1)
    for rows, cols, fmt in ((5, 70, 16), (130, 33, 32), (1, 1, 16), (129, 300, 32)):
        x = rng.standard_normal((rows, cols))
        code, byte = ref.quantize(x, fmt)
        got, gotb, clean = ref.unpack(*ref.pack(code, byte), rows, cols, fmt)
        assert clean and (got == code).all() and (gotb == byte).all()
        f = np.repeat(ref.factors(byte, fmt), fmt, 1)[:, :cols]
        # steps of e2m1 are at most 2 (from 4 to 6), and a block maximum lands at most at 8 factors (blocks of 32)
        assert (np.abs(ref.values(code, byte, fmt) - x) <= np.where(np.abs(x) > 6 * f, 2, 1) * f * (1 + 1e-12)).all()

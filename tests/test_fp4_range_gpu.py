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

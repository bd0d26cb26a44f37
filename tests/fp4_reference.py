"""4-bit matrices by their definition, in 64 bits on the CPU (numpy): what the kernels of fp4_*.cu are tested against."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# every finite e4m3 value in the order of its byte
E4M3 = np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
                 for e in range(16) for m in range(8)][:127])


def nearest(v, table):
    """Index of the entry of an ascending table nearest to v >= 0; a tie goes to the even index; the last one beyond it."""
    hi = np.minimum(np.searchsorted(table, v), len(table) - 1)
    lo = np.maximum(hi - 1, 0)
    below, above = v - table[lo], table[hi] - v
    return np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)


def factors(byte, fmt):
    byte = byte.astype(np.int64)
    if fmt == 32:
        return np.where(byte == 255, np.nan, np.ldexp(1.0, np.minimum(byte, 254) - 127))
    return np.where((byte & 127) == 127, np.nan, E4M3[np.minimum(byte & 127, 126)])


def quantize(x, fmt, scale=1.0):
    """x [rows, cols] float64 -> (codes [rows, cols] 0..15, factor bytes [rows, blocks])."""
    rows, cols = x.shape
    nb = -(-cols // fmt)
    v = np.zeros((rows, nb * fmt))
    v[:, :cols] = x / scale
    v = v.reshape(rows, nb, fmt)
    bad = ~np.isfinite(v).all(2)
    v[bad] = 0
    top = np.abs(v).max(2)
    if fmt == 16:
        byte = nearest(np.minimum(top / 6, 448.0), E4M3)
        s = E4M3[byte]
    else:
        e = np.clip(np.frexp(top)[1] - 1 - 2, -127, 127)
        e = np.where(top == 0, -127, e)
        byte, s = e + 127, np.ldexp(1.0, e)
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(s[:, :, None] > 0, np.abs(v) / s[:, :, None], 0.0)
    code = nearest(q, LEVELS) | (np.signbit(v).astype(np.int64) << 3)
    byte = np.where(bad, 255 if fmt == 32 else 127, byte)
    return code.reshape(rows, nb * fmt)[:, :cols], byte.astype(np.uint8)


def values(code, byte, fmt, scale=1.0):
    """The float64 values of codes [rows, cols] with factor bytes [rows, blocks]."""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    return v * np.repeat(factors(byte, fmt), fmt, 1)[:, :code.shape[1]] * scale


def pack(code, byte):
    """-> (codes [rows, 16 ceil(cols / 32)] uint8, factor tiles uint8), padding 0."""
    rows, cols = code.shape
    wide = np.zeros((rows, 32 * -(-cols // 32)), np.uint8)
    wide[:, :cols] = code
    nb = byte.shape[1]
    tiles, chunks = -(-rows // 128), -(-nb // 4)
    fac = np.zeros((tiles, chunks, 512), np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(nb), indexing="ij")
    fac[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4] = byte
    return wide[:, 0::2] | (wide[:, 1::2] << 4), fac.reshape(-1)


def unpack(codes, fac, rows, cols, fmt):
    """The inverse of pack; also returns whether every padding code and factor is 0."""
    codes = codes.reshape(rows, -1)
    wide = np.stack([codes & 15, codes >> 4], 2).reshape(rows, -1)
    nb = -(-cols // fmt)
    tiles, chunks = -(-rows // 128), -(-nb // 4)
    r, b = np.meshgrid(np.arange(tiles * 128), np.arange(chunks * 4), indexing="ij")
    byte = fac.reshape(tiles, chunks, 512)[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4]
    clean = not wide[:, cols:].any() and not byte[rows:].any() and not byte[:, nb:].any()
    return wide[:, :cols].astype(np.int64), byte[:rows, :nb], clean

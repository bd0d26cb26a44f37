"""What is measured of the 4-bit operators: quantising, dequantising, the product of two 4-bit matrices, and the product
of a few 16- or 32-bit rows with a 4-bit matrix.

A 4-bit matrix [rows, cols] is a pair of byte tensors. ``codes`` [rows, 16 * ceil(cols / 32)] holds two e2m1 values per
byte (sign, two exponent bits, one mantissa bit; the even column in the low half). ``scales`` holds one factor per
block of 16 columns (format 16: e4m3) or 32 columns (format 32: a power of two, stored as exponent + 127), in tiles of
128 rows x 4 blocks: byte (r % 32) * 16 + (r // 32) * 4 + b of a tile, the tiles of a row group behind one another.
A value is code * block factor * the matrix's own factor ``scale``.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"f32": 4, "f16": 2, "bf16": 2}
_LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
_handles, _tables = {}, {}


def _engine():
    """The framework and a context of the current device, as a program has them from its start on."""
    dev = torch.cuda.current_device()
    if dev not in _handles:
        name = "flux2_c_b200"
        if name not in sys.modules:
            pkg = os.path.join(os.getcwd(), "flux2.c_b200")
            spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"),
                                                          submodule_search_locations=[pkg])
            sys.modules[name] = importlib.util.module_from_spec(spec)
            spec.loader.exec_module(sys.modules[name])
        _handles[dev] = (sys.modules[name], sys.modules[name].Context(dev))
    return _handles[dev]


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token's activations on their way into a 4-bit linear of the text encoder
        {"name": "quantize one token", "op": "quantize", "rows": 1, "cols": 2560, "dtype": "bf16", "block": 16,
         "scale": 1.0, "pad": 0},
        # the feed-forward activations of one 512-token prompt
        {"name": "quantize prompt", "op": "quantize", "rows": 512, "cols": 9728, "dtype": "f16", "block": 32,
         "scale": 1.0, "pad": 0},
        # ragged f32 rows out of a wider buffer, with a factor for the whole matrix
        {"name": "quantize ragged f32", "op": "quantize", "rows": 1023, "cols": 1001, "dtype": "f32", "block": 16,
         "scale": 0.25, "pad": 7},
        # the feed-forward activations of the largest image: 8704 tokens
        {"name": "quantize image tokens", "op": "quantize", "rows": 8704, "cols": 9216, "dtype": "bf16", "block": 16,
         "scale": 1.0, "pad": 0},
        # a weight back in 16 bits, for a path that wants it so
        {"name": "dequantize weight", "op": "dequantize", "rows": 9728, "cols": 2560, "dtype": "bf16", "block": 16,
         "scale": 0.5, "pad": 0},
        # ragged, into f32
        {"name": "dequantize ragged", "op": "dequantize", "rows": 777, "cols": 1111, "dtype": "f32", "block": 32,
         "scale": 1.0, "pad": 3},
        # one token through the text encoder's down projection
        {"name": "product one token", "op": "gemm", "rows": 1, "n": 2560, "cols": 9728, "dtype": "bf16", "block": 16,
         "scale": 1.0, "residual": False},
        # one prompt through the text encoder's gate and up projections
        {"name": "product prompt", "op": "gemm", "rows": 512, "n": 19456, "cols": 2560, "dtype": "f16", "block": 32,
         "scale": 1.0, "residual": False},
        # odd sizes into the f32 residual stream, with the gate of a block
        {"name": "product ragged gated", "op": "gemm", "rows": 77, "n": 1001, "cols": 1111, "dtype": "f32", "block": 16,
         "scale": 0.5, "residual": True},
        # the largest image's tokens through a feed-forward block
        {"name": "product image tokens", "op": "gemm", "rows": 8704, "n": 18432, "cols": 9216, "dtype": "bf16",
         "block": 16, "scale": 1.0, "residual": False},
        # one token, activations kept in 16 bits
        {"name": "few rows one token", "op": "gemv", "rows": 1, "n": 19456, "cols": 2560, "dtype": "bf16", "block": 16,
         "scale": 1.0},
        # the modulation vectors of a four-step schedule in f32
        {"name": "few rows four steps", "op": "gemv", "rows": 4, "n": 18432, "cols": 9216, "dtype": "f32", "block": 32,
         "scale": 1.0},
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, min(hi, v))

    op = rng.choice(["quantize", "dequantize", "gemm", "gemm", "gemv"])
    case = {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "block": rng.choice([16, 32]),
            "scale": rng.choice([0.25, 0.5, 1.0, 2.0])}
    if op in ("quantize", "dequantize"):
        case.update(rows=size(1, 8704), cols=size(16, 9728), pad=rng.choice([0, 0, 1, 5, 8]))
    elif op == "gemm":
        case.update(rows=size(1, 8704), n=size(16, 18432), cols=size(32, 9216), residual=rng.choice([False, True]))
    else:
        case.update(rows=rng.randint(1, 16), n=size(16, 18432), cols=size(32, 9216))
    if rng.random() < 0.5:  # sizes that models have, beside odd ones
        for key in ("rows", "cols", "n"):
            if key in case and case[key] > 64:
                case[key] -= case[key] % 64
    return case


# ---------------------------------------------------------------------------------------------------- layouts
def _table(name, values, device):
    """Constants of this file on the device, in 64 bits."""
    if (name, device) not in _tables:
        _tables[name, device] = torch.tensor(values, dtype=torch.float64, device=device)
    return _tables[name, device]


def _two_to(e):
    """2^e for whole e in [-160, 127], from a table: the library's own powers may be off by a unit in the last place."""
    return _table("two to", [2.0 ** i for i in range(-160, 128)], e.device)[e.long() + 160]


def _blocks(cols, block):
    return -(-cols // block)


def _code_bytes(rows, cols):
    return rows * 16 * _blocks(cols, 32)


def _pack_scales(plain):
    """[rows, blocks] bytes -> tiles of 128 x 4."""
    rows, nb = plain.shape
    t, c = -(-rows // 128), -(-nb // 4)
    full = torch.zeros(t * 128, c * 4, dtype=torch.uint8, device=plain.device)
    full[:rows, :nb] = plain
    return full.view(t, 4, 32, c, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack_scales(scales, rows, cols, block):
    """The block factors as f32 [rows, blocks]."""
    nb = _blocks(cols, block)
    t, c = -(-rows // 128), -(-nb // 4)
    b = scales.view(t, c, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(t * 128, c * 4)[:rows, :nb]
    if block == 32:
        return torch.where(b == 255, math.nan, _two_to(b.int().clamp(max=254) - 127).float())
    e, m = ((b >> 3) & 15).int(), (b & 7).float()
    v = torch.where(e == 0, m * 2.0 ** -9, (1.0 + m / 8.0) * _two_to(e - 7).float())
    return torch.where((b & 127) == 127, math.nan, v)


def _decode(codes, scales, rows, cols, block):
    """The values of a 4-bit matrix, without its own factor, f32 [rows, cols]."""
    levels = _table("signed levels", _LEVELS + [-v for v in _LEVELS], codes.device).float()
    v = torch.stack([levels[(codes & 15).int()], levels[(codes >> 4).int()]], dim=2).view(rows, -1)
    s = _unpack_scales(scales, rows, cols, block)
    nb = s.shape[1]
    width = nb * block
    if width > v.shape[1]:
        v = torch.nn.functional.pad(v, (0, width - v.shape[1]))
    return (v[:, :width].reshape(rows, nb, block) * s[:, :, None]).view(rows, width)[:, :cols]


# ---------------------------------------------------------------------------------------------------- inputs
def _normal(shape, gen):
    return torch.randn(shape, device="cuda", generator=gen)


def _four_bit(rows, cols, block, gen, std):
    """A 4-bit matrix as quantised normal data has it."""
    nb = _blocks(cols, block)
    x = _normal((rows, nb * block), gen) * std
    x[:, cols:] = 0
    x = x.view(rows, nb, block)
    top = x.abs().amax(2)
    if block == 16:
        s8 = (top / 6).to(torch.float8_e4m3fn)
        s, plain = s8.float(), s8.view(torch.uint8)
    else:
        e = (torch.frexp(top).exponent - 3).clamp(-127, 127)
        s, plain = _two_to(e).float(), (e + 127).to(torch.uint8)
    v = (x.abs() / s[:, :, None]).nan_to_num(0.0).view(rows, nb * block)
    code = torch.bucketize(v, torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device="cuda")).to(torch.uint8)
    code |= (x.view(rows, nb * block) < 0).to(torch.uint8) << 3
    wide = 32 * _blocks(cols, 32)
    if wide > code.shape[1]:
        code = torch.nn.functional.pad(code, (0, wide - code.shape[1]))
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous(), _pack_scales(plain)


def _buffers(rows, cols, block):
    nb = _blocks(cols, block)
    return (torch.empty(_code_bytes(rows, cols), dtype=torch.uint8, device="cuda"),
            torch.empty(-(-rows // 128) * -(-nb // 4) * 512, dtype=torch.uint8, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, cols, block, dtype = case["rows"], case["cols"], case["block"], _DTYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] == "quantize":
        # activations: normal, some columns larger than the rest, as after a feed-forward block
        wide = torch.empty(rows, cols + case["pad"], dtype=dtype, device="cuda")
        big = torch.where(torch.rand(cols, device="cuda", generator=gen) < 0.01, 20.0, 1.0)
        wide[:, :cols] = _normal((rows, cols), gen) * big * case["scale"]
        st["x"], st["ld"] = wide[:, :cols], cols + case["pad"]
        st["codes"], st["scales"] = _buffers(rows, cols, block)
        st["out"] = torch.empty(rows, cols, dtype=dtype, device="cuda")
    elif case["op"] == "dequantize":
        st["codes"], st["scales"] = _four_bit(rows, cols, block, gen, 0.05)
        st["wide"] = torch.zeros(rows, cols + case["pad"], dtype=dtype, device="cuda")
        st["out"], st["ld"] = st["wide"][:, :cols], cols + case["pad"]
    else:
        n = case["n"]
        st["wcodes"], st["wscales"] = _four_bit(n, cols, block, gen, 1.0 / math.sqrt(cols))
        st["out"] = torch.empty(rows, n, dtype=dtype, device="cuda")
        if case["op"] == "gemm":
            st["codes"], st["scales"] = _four_bit(rows, cols, block, gen, 1.0)
            st["residual"] = _normal((rows, n), gen) if case["residual"] else None
            st["gate"] = _normal((n,), gen) if case["residual"] else None
        else:
            st["x"] = _normal((rows, cols), gen).to(dtype)
    return st


# ---------------------------------------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_own(st):
    fx, ctx = _engine()
    c = st["case"]
    dtype = {"f32": fx.F32, "f16": fx.F16, "bf16": fx.BF16}[c["dtype"]]
    rows, cols, block = c["rows"], c["cols"], c["block"]
    out = st["out"]
    if c["op"] == "quantize":
        q = fx.Fp4(st["codes"].data_ptr(), st["scales"].data_ptr(), rows, cols, block, c["scale"])
        ctx.fp4_quantize(st["x"].data_ptr(), dtype, st["ld"], q)
        ctx.fp4_dequantize(q, out.data_ptr(), dtype, cols)
    elif c["op"] == "dequantize":
        q = fx.Fp4(st["codes"].data_ptr(), st["scales"].data_ptr(), rows, cols, block, c["scale"])
        ctx.fp4_dequantize(q, out.data_ptr(), dtype, st["ld"])
    else:
        w = fx.Fp4(st["wcodes"].data_ptr(), st["wscales"].data_ptr(), c["n"], cols, block, c["scale"])
        if c["op"] == "gemm":
            x = fx.Fp4(st["codes"].data_ptr(), st["scales"].data_ptr(), rows, cols, block, 1.0)
            if st["residual"] is None:
                ctx.gemm_fp4(x, w, out.data_ptr(), dtype, c["n"])
            else:
                ctx.gemm_fp4(x, w, out.data_ptr(), dtype, c["n"], gate_ptr=st["gate"].data_ptr(),
                             residual_ptr=st["residual"].data_ptr(), ld_residual=c["n"])
        else:
            ctx.gemv_fp4(st["x"].data_ptr(), dtype, cols, rows, w, out.data_ptr(), dtype, c["n"])
    return out


def _round_e4m3(v):
    """Non-negative values to the nearest e4m3 value, ties to even, at most 448; in 64 bits, since a third of a 32-bit
    number may lie next to a border."""
    e = (torch.frexp(v).exponent - 1).clamp(min=-6)
    step = _two_to(e - 3)
    return (torch.round(v / step) * step).clamp(max=448.0)


def _block_scales(top, block):
    if block == 16:
        six = torch.full((), 6.0, dtype=torch.float64, device=top.device)  # a plain 6 would become a product with 1 / 6
        s = _round_e4m3(top.double() / six).float()
    else:
        s = _two_to((torch.frexp(top).exponent - 3).clamp(-127, 127)).float()
    return torch.where(torch.isfinite(top), s, math.nan)


def _run_plain(st):
    c = st["case"]
    rows, cols, block, dtype = c["rows"], c["cols"], c["block"], _DTYPES[c["dtype"]]
    if c["op"] == "quantize":
        nb = _blocks(cols, block)
        x = torch.nn.functional.pad(st["x"].float() / c["scale"], (0, nb * block - cols)).view(rows, nb, block)
        s = _block_scales(x.abs().amax(2), block)[:, :, None]
        v = torch.where(s == 0, 0.0, x / s)  # the quotient of a short factor is never rounded onto a border
        a = v.abs()
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        q = (torch.round(a / step) * step).clamp(max=6.0) * torch.sign(v)
        return (q * s * c["scale"]).view(rows, nb * block)[:, :cols].to(dtype)
    if c["op"] == "dequantize":
        return (_decode(st["codes"], st["scales"], rows, cols, block) * c["scale"]).to(dtype)
    w = _decode(st["wcodes"], st["wscales"], c["n"], cols, block)
    if c["op"] == "gemv":
        return (st["x"].float() @ w.t() * c["scale"]).to(dtype)
    y = _decode(st["codes"], st["scales"], rows, cols, block) @ w.t() * c["scale"]
    if st["residual"] is not None:
        y = st["residual"] + st["gate"] * y
    return y.to(dtype)


# ---------------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    rows, cols, block, size = case["rows"], case["cols"], case["block"], _SIZES[case["dtype"]]

    def packed(r):
        return _code_bytes(r, cols) + r * _blocks(cols, block)

    if case["op"] == "quantize":  # the values are read, the codes written, and the values that they stand for
        return {"bytes": rows * cols * 2 * size + packed(rows), "flops": 0}
    if case["op"] == "dequantize":
        return {"bytes": rows * cols * size + packed(rows), "flops": 0}
    n = case["n"]
    bytes_ = packed(n) + rows * n * size
    if case["op"] == "gemm":
        bytes_ += packed(rows) + ((rows * n + n) * 4 if case["residual"] else 0)
    else:
        bytes_ += rows * cols * size
    return {"bytes": bytes_, "flops": 2.0 * rows * n * cols}


# ---------------------------------------------------------------------------------------------------- from the definition, in 64 bits
def _nearest(v, table):
    """v >= 0 to the nearest entry of an ascending table, a tie to the entry of even index, the last one beyond it."""
    hi = torch.searchsorted(table, v).clamp(max=table.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    below, above = v - table[lo], table[hi] - v
    take_lo = (below < above) | ((below == above) & (lo % 2 == 0))
    return torch.where(take_lo, table[lo], table[hi])


def _values64(codes, scales, rows, cols, block, first, last):
    """Rows [first, last) of a 4-bit matrix, in 64 bits, column by column from the layout's own formula."""
    dev = codes.device
    r = torch.arange(first, last, device=dev)[:, None]
    k = torch.arange(cols, device=dev)[None, :]
    byte = codes.reshape(rows, -1)[first:last][:, torch.arange(cols, device=dev) // 2].long()
    code = torch.where(k % 2 == 1, byte >> 4, byte & 15)
    mag = code & 7
    exp, man = mag >> 1, (mag & 1).double()
    v = torch.where(exp == 0, man * 0.5, (1 + man / 2) * _two_to(exp - 1))
    v = torch.where(code >= 8, -v, v)
    chunks = -(-_blocks(cols, block) // 4)
    b = torch.arange(_blocks(cols, block), device=dev)[None, :]
    at = ((r // 128) * chunks + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
    s = scales.reshape(-1)[at].long()
    if block == 32:
        f = _two_to(s - 127)
    else:
        e, m = s >> 3 & 15, (s & 7).double() / 8
        f = torch.where(e == 0, m * 2.0 ** -6, (1 + m) * _two_to(e - 7))
    return v * f.repeat_interleave(block, 1)[:, :cols]


def exact(case, seed):
    st = prepare(case, seed)
    rows, cols, block = case["rows"], case["cols"], case["block"]
    if case["op"] == "quantize":
        dev = st["x"].device
        levels = _table("levels", _LEVELS, dev)
        if block == 16:
            bits = torch.arange(127, device=dev)
            e, m = bits >> 3, (bits & 7).double() / 8
            table = torch.where(e == 0, m * 2.0 ** -6, (1 + m) * _two_to(e - 7))
        else:
            table = _two_to(torch.arange(-149, 128, device=dev))
        nb, out = _blocks(cols, block), []
        for a in range(0, rows, 512):
            x = st["x"][a:a + 512].double() / case["scale"]
            x = torch.cat([x, x.new_zeros(x.shape[0], nb * block - cols)], 1)
            top = x.abs().view(-1, nb, block).max(2).values
            if block == 16:
                s = _nearest(top / torch.full_like(top, 6.0), table)
            else:
                below = table[(torch.searchsorted(table, top, right=True) - 1).clamp(min=0)]
                s = (below / 4).clamp(min=2.0 ** -127)
            s = s.repeat_interleave(block, 1)
            q = torch.where(s > 0, _nearest((x.abs() / s).nan_to_num(0.0, 0.0), levels), 0.0)
            out.append((q * torch.sign(x) * s * case["scale"])[:, :cols])
        return torch.cat(out)
    if case["op"] == "dequantize":
        return torch.cat([_values64(st["codes"], st["scales"], rows, cols, block, a, min(a + 512, rows))
                          for a in range(0, rows, 512)]) * case["scale"]
    x = st["x"].double() if case["op"] == "gemv" else _values64(st["codes"], st["scales"], rows, cols, block, 0, rows)
    n = case["n"]
    y = torch.empty(rows, n, dtype=torch.float64, device=x.device)
    for a in range(0, n, 1024):
        w = _values64(st["wcodes"], st["wscales"], n, cols, block, a, min(a + 1024, n))
        y[:, a:a + 1024] = torch.einsum("mk,nk->mn", x, w)
    y *= case["scale"]
    if case["op"] == "gemm" and case["residual"]:
        y = st["residual"].double() + st["gate"].double() * y
    return y

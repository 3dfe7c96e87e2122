"""Performance cases of the microscaled forms: what a served model keeps and multiplies by, in 4 or
8 bits with a power-of-two scale for every 32 values along the last axis.

`kernels.mx_quantise` and `kernels.mx_dequantise` write and read them, `kernels.mx_linear` is a
projection with a 4-bit weight and 4-bit activations, and `kernels.refresh_capture` writes a
refinement bank in 8 bits.  Shapes are those of the benchmark's videos, of the tests, and generic
sizes between them.

A block of 32 values whose largest magnitude is a has the scale 2^e:
    "fp4"    e the smallest with a < 7 * 2^e; values on 0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^e
    "int8"   e the smallest with 64 * a < 127.5 * 2^e; values on integers up to 127 times 2^(e - 6)
both to the nearest, ties to the even code.  Scales are held as e + 127 in a byte; rows of "fp4" are
filled up with zeros to 256 values, two to a byte, the first in the low half.

A case is a dict of plain values.
kind "quantise": rows, width, dtype, format, source: the rows as they are written, then read back
    ("rows": contiguous; "part": the middle third of rows three times as wide)
kind "dequantise": rows, width, dtype, format: kept codes read back as dtype
kind "linear": rows, width (in), outputs, dtype, out (type of the result), bias,
    kept (whether the activations are codes already, as for the second of two projections)
kind "capture": heads, dim, frames, height, width, text, text_first, dtype: a layer's refinement
    written into its bank; the bank's values and log-masses
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK, FP4_ROW = 32, 256
MAX_VALUES = 24 * 128 * 118784             # of one quantised tensor, the largest bank's
MAX_PRODUCT = 118800 * 2048 * 8192         # multiplications of the largest projection
MAX_RESULT = 118800 * 8192


def _quantise(name, rows, width, format, *, dtype="bf16", source="rows"):
    case = dict(kind="quantise", rows=rows, width=width, dtype=dtype, format=format, source=source)
    return case if name is None else dict(case, name=name)


def _dequantise(name, rows, width, format, *, dtype="bf16"):
    case = dict(kind="dequantise", rows=rows, width=width, dtype=dtype, format=format)
    return case if name is None else dict(case, name=name)


def _linear(name, rows, width, outputs, *, dtype="bf16", out=None, bias=True, kept=False):
    case = dict(kind="linear", rows=rows, width=width, outputs=outputs, dtype=dtype,
                out=out or dtype, bias=bias, kept=kept)
    return case if name is None else dict(case, name=name)


def _capture(name, heads, dim, frames, height, width, *, text=0, text_first=False, dtype="bf16"):
    case = dict(kind="capture", heads=heads, dim=dim, frames=frames, height=height, width=width,
                text=text, text_first=text_first, dtype=dtype)
    return case if name is None else dict(case, name=name)


def listed():
    return [
        # A prompt's text stream before its projections: few rows, latency counts.
        _quantise("quantise-text", 256, 2048, "fp4", dtype="fp16"),
        # The 480p stream before a block's projections.
        _quantise("quantise-480p", 21 * 30 * 52, 1536, "fp4"),
        # An fp16 refinement of the 720p video, kept in 8 bits from here on.
        _quantise("quantise-bank-720p", 24 * 118784, 128, "int8", dtype="fp16"),
        # A projection's weight of odd sizes, read back for a layer that has to have it in fp32.
        _dequantise("read-weight-odd", 1155, 1155, "fp4", dtype="fp32"),
        # The 480p video's refinement, read back whole.
        _dequantise("read-bank-480p", 12 * 255 * 128, 128, "int8", dtype="fp16"),
        # A timestep's scales, shifts and gates for a guided pair: two rows, six vectors.
        _linear("linear-timestep", 2, 1536, 6 * 1536, out="fp32"),
        # The text stream's projection.
        _linear("linear-text", 256, 2048, 2048, dtype="fp16"),
        # The 480p stream's keys, its activations in 4 bits from the queries' projection.
        _linear("linear-480p-kept", 21 * 30 * 52, 1536, 1536, kept=True),
        # Odd sizes on every side, no bias.
        _linear("linear-odd", 15876, 1155, 999, bias=False),
        # The 720p stream into a feed-forward block: the largest product.
        _linear("linear-720p", 33 * 45 * 80, 2048, 8192),
        # The bank of a thumbnail clip's two heads: launches, where latency counts.
        _capture("capture-thumbnail", 2, 64, 4, 32, 32),
        # The 720p video's bank with its text tokens last.
        _capture("capture-720p", 24, 128, 33, 45, 80, text=256),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A width: two of three are multiples of 32, the others anything."""
    n = _log_int(rng, lo, hi)
    return max(32, n // 32 * 32) if rng.random() < 0.67 else n


def _draw_rows(rng, kind):
    """One row to a 720p bank, widths from one block to 8192."""
    while True:
        rows, width = _log_int(rng, 1, 24 * 118784), _size(rng, 32, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        format = rng.choice(["fp4", "int8"])
        source = rng.choice(["rows", "part"]) if kind == "quantise" else "rows"
        weight = (2 if dtype == "fp32" else 1) * (3 if source == "part" else 1)
        filled = -(-width // FP4_ROW) * FP4_ROW if format == "fp4" else width
        if rows * filled * weight <= MAX_VALUES:
            return _quantise(None, rows, width, format, dtype=dtype, source=source) \
                if kind == "quantise" else _dequantise(None, rows, width, format, dtype=dtype)


def _draw_linear(rng):
    """One row to a 720p video, any widths on both sides."""
    while True:
        rows, width, outputs = _log_int(rng, 1, 118800), _size(rng, 64, 8192), _size(rng, 64, 8192)
        if rows * width * outputs <= MAX_PRODUCT and rows * max(width, outputs) <= MAX_RESULT:
            dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
            return _linear(None, rows, width, outputs, dtype=dtype,
                           out=rng.choice([dtype, dtype, "fp32"]), bias=rng.random() < 0.6,
                           kept=rng.random() < 0.4)


def _draw_capture(rng):
    """From one block of 128 tokens to 720p, 1 to 48 heads, both head sizes."""
    while True:
        frames = rng.randint(1, 33)
        side = math.sqrt(math.exp(rng.uniform(math.log(160), math.log(118800))) / frames)
        aspect = rng.uniform(0.5, 1.0)
        height, width = max(1, int(side * aspect ** 0.5)), max(1, int(side / aspect ** 0.5))
        dim, heads = rng.choice([64, 128]), _log_int(rng, 1, 48)
        tokens = frames * height * width
        if tokens >= 128 and heads * dim * tokens <= MAX_VALUES:
            return _capture(None, heads, dim, frames, height, width,
                            text=rng.choice([0, 77, 226, 256, rng.randint(1, 300)]),
                            text_first=rng.random() < 0.5,
                            dtype="fp16" if rng.random() < 0.3 else "bf16")


def draw(rng):
    kind = rng.choice(["quantise", "dequantise", "linear", "linear", "capture"])
    if kind == "linear":
        return _draw_linear(rng)
    return _draw_capture(rng) if kind == "capture" else _draw_rows(rng, kind)


# -- the plain forms -----------------------------------------------------------------------

# Exponent of a format's largest power of two, the mantissa in [0.5, 1) from which the largest
# value would round past the largest code, and that code.
_PLAIN = {"fp4": (2, 7 / 8, 6.0), "int8": (6, 255 / 256, 127.0)}


def _plain_values(x, format):
    """(values on the format's grid, exponent of a value of one) of fp32 blocks [..., 32]."""
    top, past, largest = _PLAIN[format]
    mantissa, exponent = torch.frexp(x.abs().amax(-1, keepdim=True))
    shift = exponent - 1 - top + (mantissa >= past).to(torch.int32)
    shift = shift.clamp(min=-127 - (top if format == "int8" else 0))
    v = torch.ldexp(x, -shift)
    if format == "fp4":
        size = v.abs()
        step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
        v = torch.copysign(torch.round(size / step) * step, x)
    else:
        v = torch.round(v)
    return v.clamp(-largest, largest), shift


def _blocks(x, fill=BLOCK):
    """fp32 rows [rows, width] as blocks [rows, blocks, 32], zeros behind the width."""
    x = torch.nn.functional.pad(x.float(), (0, -x.shape[1] % fill))
    return x.unflatten(1, (-1, BLOCK))


def _plain_rounded(x, format):
    """fp32 rows rounded to what their microscaled form holds."""
    v, shift = _plain_values(_blocks(x), format)
    return torch.ldexp(v, shift).flatten(1)[:, :x.shape[1]]


def _codes(x, format):
    """(codes, scales) of fp32 rows as they are kept."""
    v, shift = _plain_values(_blocks(x, FP4_ROW if format == "fp4" else BLOCK), format)
    scales = (shift + (127 if format == "fp4" else 133)).squeeze(-1).to(torch.uint8)
    v = v.flatten(1)
    if format == "int8":
        return v.to(torch.int8), scales
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=x.device)
    code = torch.bucketize(v.abs(), grid).to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)
    return code[:, ::2] + 16 * code[:, 1::2], scales


def _plain_read(codes, scales, format, width):
    """fp32 values of kept rows."""
    if format == "int8":
        v, shift = codes.float(), scales.to(torch.int32) - 133
    else:
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
        grid = torch.cat([grid, -grid])
        v = grid[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(1).int()]
        shift = scales.to(torch.int32) - 127
    return torch.ldexp(v.unflatten(1, (-1, BLOCK)), shift.unsqueeze(-1)).flatten(1)[:, :width]


def _plain_capture(state):
    s, rows = state, state["rows"]
    at = s["rowmap"][:rows].long()
    lf, of = s["dense_lse"][0][:, at], s["dense_out"][0][:, at].float()
    lh, oh = s["head_lse"][:, :rows], s["head_out"][:, :rows].float()
    # In 64 bits: in 32 what the kept blocks leave of a row, 1 - ratio, is lost beside it.
    lf, lh = lf.double(), lh.double()
    ratio = torch.exp((lh - lf).clamp(max=0)).clamp(max=1 - 1e-6)
    rest = 1 - ratio
    tail = (of - ratio[..., None].float() * oh) / rest[..., None].float()
    detail = (tail - s["go"].float()).clamp(-6e4, 6e4)
    detail = torch.where(ratio[..., None] > 1 - 1e-3, 0.0, detail)
    value = _plain_rounded(detail.flatten(0, 1), "int8").view_as(detail)
    mass = (lf + torch.log(rest) - s["gl"].double()).clamp(-30, 30)
    return value.to(torch.float16), mass.float()


def _plain(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "capture":
        return _plain_capture(state)
    if kind == "quantise":
        return _plain_rounded(state["x"], case["format"]).to(DTYPES[case["dtype"]])
    if kind == "dequantise":
        return _plain_read(state["codes"], state["scales"], case["format"],
                           case["width"]).to(DTYPES[case["dtype"]])
    width = case["width"]
    x = _plain_read(*state["x"], "fp4", width) if case["kept"] else \
        _plain_rounded(state["x"], "fp4")
    y = x @ _plain_read(*state["weight"], "fp4", width).T
    if case["bias"]:
        y = y + state["bias"].float()
    return y.to(DTYPES[case["out"]])


# -- what a program holds before the call --------------------------------------------------


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def _channels(g, width, spread):
    """Per-channel sizes as trained layers have them: most near one, a few large."""
    size = torch.exp(spread * _normal(g, width))
    return torch.where(torch.rand(width, generator=g, device="cuda") < 0.01, 6 * size, size)


def _rows(g, rows, width, dtype):
    return _normal(g, rows, width, dtype=dtype).mul_(_channels(g, width, 0.4).to(dtype))


def _kept_rows(g, rows, width, format):
    """(codes, scales) of rows, a part of them at a time."""
    size = _channels(g, width, 0.4)
    step = max(1, (1 << 27) // (-(-width // FP4_ROW) * FP4_ROW))
    parts = [_codes(_normal(g, min(step, rows - first), width) * size, format)
             for first in range(0, rows, step)]
    return tuple(torch.cat(p) if len(p) > 1 else p[0] for p in zip(*parts))


def _row_order(frames, height, width):
    """Video tokens in the order of boxes of 4 x 4 x 8, as blocks of 128 neighbours have them."""
    at = torch.arange(frames * height * width, device="cuda")
    t, y, x = at // (height * width), at // width % height, at % width
    box = (t // 4 * (height // 4 + 1) + y // 4) * (width // 8 + 1) + x // 8
    return torch.argsort(box * 128 + (t % 4 * 4 + y % 4) * 8 + x % 8)


def _prepare_capture(case, g):
    """A layer at a refresh: the dense output, the kept blocks' and the coarse tail's, as their
    masses make it from two parts."""
    h, d, dtype = case["heads"], case["dim"], DTYPES[case["dtype"]]
    video = case["frames"] * case["height"] * case["width"]
    n, rows = video + case["text"], video // 128 * 128
    first = case["text"] if case["text_first"] else 0
    order = _row_order(case["frames"], case["height"], case["width"]) + first
    text = torch.arange(case["text"], device="cuda") + (0 if case["text_first"] else video)
    rowmap = torch.cat([order, text]).to(torch.int32)
    ratio = 0.25 + 0.7 * torch.rand(h, n, generator=g, device="cuda")
    ratio[:, ::61] = 0.9996  # rows whose kept blocks are all that counts
    head = 0.3 * _normal(g, h, n, d, dtype=dtype)
    go = 0.2 * _normal(g, h, rows, d, dtype=dtype)
    detail = _normal(g, h, rows, d, dtype=dtype).mul_((0.1 * _channels(g, d, 0.5)).to(dtype))
    dense = head.clone()
    share = ratio[:, :rows, None].to(dtype)
    dense[:, :rows].mul_(share).add_((1 - share) * (detail + go))
    back = torch.argsort(rowmap.long())
    lse = 9 + 0.5 * _normal(g, h, n)
    rest = torch.log1p(-ratio[:, :rows])
    return dict(case=case, rows=rows, video=video, rowmap=rowmap, dense_out=dense[None, :, back],
                dense_lse=lse[None, :, back].contiguous(), head_out=head,
                head_lse=lse + torch.log(ratio), go=go,
                gl=lse[:, :rows] + rest + 0.3 * _normal(g, h, rows),
                codes=torch.zeros(h, rows, d, dtype=torch.int8, device="cuda"),
                scales=torch.zeros(h, rows, d // BLOCK, dtype=torch.uint8, device="cuda"),
                mass=torch.zeros(h, rows, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, width = case["kind"], case.get("width")
    if kind == "capture":
        return _prepare_capture(case, g)
    dtype, state = DTYPES[case["dtype"]], dict(case=case)
    if kind == "dequantise":
        state["codes"], state["scales"] = _kept_rows(g, case["rows"], width, case["format"])
    elif kind == "quantise" and case["source"] == "part":
        state["x"] = _rows(g, case["rows"], 3 * width, dtype)[:, width:2 * width]
    elif kind == "linear" and case["kept"]:
        state["x"] = _kept_rows(g, case["rows"], width, "fp4")
    else:
        state["x"] = _rows(g, case["rows"], width, dtype)
    if kind == "linear":
        state["weight"] = _codes(_normal(g, case["outputs"], width) / math.sqrt(width), "fp4")
        if case["bias"]:
            state["bias"] = (0.2 * _normal(g, case["outputs"])).to(dtype)
    return state


# -- the framework's calls -----------------------------------------------------------------


def _own(state):
    from recap_amd import kernels

    case = state["case"]
    kind = case["kind"]
    if kind == "capture":
        geometry = kernels.Geometry(n_tokens=state["rowmap"].numel(), n_video=state["video"])
        bank = kernels.Microscaled(state["codes"], state["scales"], "int8", case["dim"])
        kernels.refresh_capture(state["dense_out"], state["dense_lse"], state["head_out"],
                                state["head_lse"], state["go"], state["gl"], state["rowmap"],
                                geometry, bank, state["mass"])
        return kernels.mx_dequantise(bank, torch.float16), state["mass"]
    dtype, width = DTYPES[case["dtype"]], case["width"]
    if kind == "quantise":
        return kernels.mx_dequantise(kernels.mx_quantise(state["x"], case["format"]), dtype)
    if kind == "dequantise":
        kept = kernels.Microscaled(state["codes"], state["scales"], case["format"], width)
        return kernels.mx_dequantise(kept, dtype)
    x = kernels.Microscaled(*state["x"], "fp4", width) if case["kept"] else state["x"]
    return kernels.mx_linear(x, kernels.Microscaled(*state["weight"], "fp4", width),
                             state.get("bias"), dtype=DTYPES[case["out"]])


def run(state):
    return _own(state) if own else _plain(state)


# -- what a pass cannot do without ---------------------------------------------------------


def _bytes(name):
    return 4 if name == "fp32" else 2


def _kept_bytes(rows, width, format):
    return rows * (width * (0.5 if format == "fp4" else 1) + -(-width // BLOCK))


def work(case):
    kind, dtype = case["kind"], _bytes(case["dtype"])
    if kind == "capture":
        video = case["frames"] * case["height"] * case["width"]
        rows = case["heads"] * (video // 128 * 128)
        kept = _kept_bytes(rows, case["dim"], "int8")
        # three tensors and three masses in, the bank out; the bank read back as fp16
        return {"bytes": rows * case["dim"] * (3 * dtype + 2) + 2 * kept + rows * 16,
                "flops": 14 * rows * case["dim"]}
    rows, width = case["rows"], case["width"]
    if kind == "linear":
        outputs = case["outputs"]
        x = _kept_bytes(rows, width, "fp4") if case["kept"] else rows * width * dtype
        return {"bytes": x + _kept_bytes(outputs, width, "fp4") + rows * outputs * _bytes(case["out"])
                + (outputs * dtype if case["bias"] else 0), "flops": 2 * rows * width * outputs}
    kept, values = _kept_bytes(rows, width, case["format"]), rows * width
    if kind == "dequantise":
        return {"bytes": kept + values * dtype, "flops": values}
    return {"bytes": 2 * values * dtype + 2 * kept, "flops": 6 * values}


# -- the definitions in 64 bits ------------------------------------------------------------


def _exact_rounded(x, format):
    """64-bit rows on the nearest values of their format, a part of the rows at a time."""
    rows, width = x.shape
    step = max(1, (1 << 27) // width)
    if rows > step:
        return torch.cat([_exact_rounded(x[i:i + step], format) for i in range(0, rows, step)])
    filled = torch.zeros(rows, -(-width // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    filled[:, :width] = x
    filled = filled.view(rows, -1, BLOCK)
    limit = 7.0 if format == "fp4" else 127.5 / 64
    largest = filled.abs().max(-1, keepdim=True).values
    unit = 2.0 ** torch.frexp(largest / limit).exponent.clamp(min=-127).double()
    v = filled / unit
    if format == "int8":
        v = torch.round(64 * v) / 64
    else:
        # The k-th border lies between the codes k and k + 1; on it the even code counts.
        borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64,
                               device=x.device)
        grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=x.device)
        below = torch.bucketize(v.abs(), borders)
        above = torch.bucketize(v.abs(), borders, right=True)
        v = torch.sign(v) * grid[torch.where(below % 2 == 0, below, above)]
    return (v * unit).view(rows, -1)[:, :width]


def _exact_read(codes, scales, format, width):
    rows = codes.shape[0]
    if format == "int8":
        v, point = codes.double(), 64.0
    else:
        nibbles = torch.empty(rows, 2 * codes.shape[1], dtype=torch.int64, device=codes.device)
        nibbles[:, 0::2], nibbles[:, 1::2] = codes % 16, codes // 16
        power, odd = nibbles // 2 % 4, nibbles % 2
        size = torch.where(power == 0, 0.5 * odd, 2.0 ** (power - 1.0) * (1 + 0.5 * odd))
        v, point = torch.where(nibbles >= 8, -size, size).double(), 1.0
    unit = 2.0 ** (scales.double() - 127) / point
    return (v.view(rows, -1, BLOCK) * unit[:, :, None]).view(rows, -1)[:, :width]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantise":
        return _exact_rounded(state["x"].double(), case["format"])
    if kind == "dequantise":
        return _exact_read(state["codes"], state["scales"], case["format"], case["width"])
    if kind == "linear":
        x = _exact_read(*state["x"], "fp4", case["width"]) if case["kept"] else \
            _exact_rounded(state["x"].double(), "fp4")
        weight = _exact_read(*state["weight"], "fp4", case["width"])
        return torch.nn.functional.linear(
            x, weight, state["bias"].double() if case["bias"] else None)
    rows = state["rows"]
    where = state["rowmap"][:rows].to(torch.int64)
    value, mass = [], []
    for head in range(case["heads"]):
        of = state["dense_out"][0, head].double()[where]
        lf = state["dense_lse"][0, head].double()[where]
        share = torch.exp(torch.minimum(state["head_lse"][head, :rows].double() - lf,
                                        torch.zeros_like(lf)))
        share = torch.minimum(share, torch.full_like(share, 1 - 1e-6))
        oh = state["head_out"][head, :rows].double()
        tail = (of - share[:, None] * oh) / (1 - share)[:, None]
        detail = torch.clamp(tail - state["go"][head].double(), -6e4, 6e4)
        detail[share > 1 - 1e-3] = 0
        value.append(_exact_rounded(detail, "int8"))
        mass.append(torch.clamp(lf + torch.log1p(-share) - state["gl"][head].double(), -30, 30))
    return torch.stack(value), torch.stack(mass)

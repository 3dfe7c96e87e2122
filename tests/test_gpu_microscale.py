"""Microscaled rows and their product on the GPU against the definitions in 64 bits: every code and
scale equal, every value read back exact, every product within half a step and the bound of its
fp32 sum; sizes from one value up, strides, alignments, extremes, streams and graphs."""

import pytest
import torch

import mx_util as M
from recap_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
FORMATS = ("fp4", "int8")


def make(seed, *shape, dtype=BF, spread=1.0):
    """Values whose channels differ in size, some of them on the borders between codes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(*shape, generator=g, device="cuda")
    x = x * (spread * torch.randn(shape[-1], generator=g, device="cuda")).exp()
    ties = torch.rand(*shape, generator=g, device="cuda") < 0.2
    return torch.where(ties, torch.round(4 * x) / 4, x).to(dtype)


def check_rows(x, format, label):
    print(f"case {label} {format} {tuple(x.shape)} {x.dtype}", flush=True)
    index, negative, byte = M.quantise(x, format)
    m = K.mx_quantise(x, format)
    assert m.shape == x.shape and m.format == format
    assert torch.equal(m.scales.cpu(), byte), f"{label}: scales"
    codes = m.codes.cpu()
    # a zero's sign is the value's own in fp4; int8 has one zero
    assert torch.equal(codes, M.pack(index, negative, format).view_as(codes)), f"{label}: codes"
    want = M.values(index, negative, byte, format, x.shape[-1])
    for dtype in (BF, FP, F32):
        got = K.mx_dequantise(m, dtype)
        assert got.dtype == dtype
        assert torch.equal(got.cpu(), want.to(dtype)), f"{label}: values in {dtype}"
    return m


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=str)
@pytest.mark.parametrize("width", [1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 100, 128, 255, 256, 257, 511,
                                   520, 1000, 1024, 1155, 1536, 2048, 4099, 8192, 8200, 20001])
def test_widths(cuda, width, dtype, format):
    check_rows(make(1, 5, width, dtype=dtype), format, "width")


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("shape", [(64,), (1, 256), (3, 0, 64), (0, 32), (2, 3, 5, 96), (257, 64),
                                   (1031, 128), (7, 1, 9, 40), (40000, 33)])
def test_shapes(cuda, shape, format):
    check_rows(make(2, *shape), format, "shape")


@pytest.mark.parametrize("format", FORMATS)
def test_every_half_step(cuda, format):
    """All multiples of a quarter code step over two binades of every sign, with a block's largest
    value at both sides of the border where the scale changes."""
    edge = M.LIMIT[format]
    step = 0.125 if format == "fp4" else 1 / 256
    base = torch.arange(0, edge + step / 2, step, dtype=torch.float64)
    rows = []
    for top in (edge, edge * (1 - 2.0 ** -23), edge * (1 + 2.0 ** -22), edge / 2, 1.0):
        v = torch.cat([base, -base])
        v = v[v.abs() <= top]
        v = torch.cat([v, torch.zeros(-v.numel() % 31)]).view(-1, 31)
        rows.append(torch.cat([torch.full((v.shape[0], 1), top), v], dim=1))
    x = torch.cat(rows).float().cuda()
    for power in (0, -30, 60):
        check_rows(torch.ldexp(x, torch.tensor(power, device="cuda")), format, f"2^{power}")


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("dtype", [BF, FP, F32], ids=str)
def test_extremes(cuda, dtype, format):
    """Zeros, subnormals, the largest values, infinities and NaN, each in blocks of their own."""
    info = torch.finfo(dtype)
    small, big = float(info.smallest_normal), float(info.max)
    parts = [[0.0], [-0.0, 0.0], [small], [small, 0.75 * small, -small / 2],
             [small / 2, small / 8], [info.eps * small], [big, 1.0, -1.0], [-big, big / 2, big / 64],
             [big / 128, -big / 3], [float("inf"), 1.0], [-float("inf")], [float("nan"), 2.0],
             [float("nan"), float("inf")], [1.0, small], [3 * small, 1.5 * small, 7 * small]]
    x = torch.zeros(len(parts), 64, dtype=F32)
    for i, part in enumerate(parts):
        x[i, 3:3 + len(part)] = torch.tensor(part)
        x[i, 40] = 0.3  # the next block is an ordinary one
    x = x.to(dtype).cuda()
    index, negative, byte = M.quantise(x, format)
    m = K.mx_quantise(x, format)
    assert torch.equal(m.scales.cpu(), byte)
    assert torch.equal(m.codes.cpu(), M.pack(index, negative, format))
    want = M.values(index, negative, byte, format, 64)
    for out in (BF, FP, F32):
        got = K.mx_dequantise(m, out).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got[ok], want.to(out)[ok]), out


@pytest.mark.parametrize("format", FORMATS)
def test_every_code_reads_exactly(cuda, format):
    """All codes under all scales, in types that hold them."""
    codes = torch.arange(-127, 128).to(torch.int8) if format == "int8" else torch.arange(256).to(torch.uint8)
    scales = torch.arange(256).to(torch.uint8)
    per = 32 if format == "int8" else 128
    row = torch.cat([codes, torch.zeros(-codes.numel() % per, dtype=codes.dtype)])
    blocks = row.numel() // (32 if format == "int8" else 16)
    width = row.numel() * (1 if format == "int8" else 2)
    m = K.Microscaled(row.expand(256, -1).contiguous().cuda(),
                      scales[:, None].expand(-1, blocks).contiguous().cuda(), format, width)
    want = M.read(m)
    for dtype in (BF, FP, F32):
        got = K.mx_dequantise(m, dtype).cpu()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert torch.equal(got[ok], want[ok].to(dtype)), dtype


@pytest.mark.parametrize("format", FORMATS)
@pytest.mark.parametrize("width", [64, 100, 768])
def test_strides_and_outputs(cuda, width, format):
    """Slices at odd offsets, transposed and expanded rows; outputs in place and beside others."""
    wide = make(3, 6, 5, 3 * width + 3)
    for x in (wide[..., 1:1 + width], wide[:, 2:4, 3:3 + width], wide.transpose(0, 1)[..., :width],
              wide[:1, :1, 2:2 + width].expand(4, 5, width), wide[0, 0, :width],
              make(4, width, 6).t()):
        m = check_rows(x, format, "view")
        again = K.Microscaled.empty(x.shape, format, "cuda")
        assert K.mx_quantise(x, format, out=again) is again
        assert torch.equal(again.codes, m.codes) and torch.equal(again.scales, m.scales)
    m = K.mx_quantise(wide[..., :width].contiguous(), format)
    for dtype in (BF, F32):
        frame = torch.full((6, 5, width + 5), 7.0, dtype=dtype, device="cuda")
        out = frame[..., 3:3 + width]
        assert K.mx_dequantise(m, dtype, out=out) is out
        assert torch.equal(out, K.mx_dequantise(m, dtype))
        assert (frame[..., :3] == 7).all() and (frame[..., 3 + width:] == 7).all()


# Sizes around every tile's, one row and one output up.
PRODUCTS = [(1, 1, 1), (1, 32, 1), (2, 64, 3), (1, 256, 64), (3, 257, 5), (5, 100, 33), (16, 512, 16),
            (17, 512, 31), (31, 300, 64), (33, 1024, 65), (64, 768, 127), (65, 256, 128), (127, 520, 129),
            (128, 1536, 128), (129, 300, 257), (200, 2048, 96), (255, 1155, 256), (257, 64, 255),
            (300, 1300, 520), (1000, 512, 300), (4, 4096, 1000), (8, 8192, 70), (1, 8192, 2000),
            (520, 2500, 1030), (16, 4200, 70), (16, 8192, 40), (9, 5000, 33), (7, 20001, 65),
            (8, 65, 10300), (16, 3841, 32)]


@pytest.mark.parametrize("rows,width,outputs", PRODUCTS)
@pytest.mark.parametrize("dtype,out", [(BF, BF), (FP, F32), (F32, F32), (BF, FP)], ids=str)
def test_products(cuda, rows, width, outputs, dtype, out):
    print(f"case {rows} {width} {outputs}", flush=True)
    x, w = make(5, rows, width, dtype=dtype, spread=0.5), make(6, outputs, width, dtype=F32, spread=0.5)
    weight = K.mx_quantise(w / width ** 0.5)
    bias = make(7, outputs, dtype=dtype)
    xq, wq = M.rounded(x, "fp4"), M.read(weight)
    got = K.mx_linear(x, weight, bias, dtype=out)
    assert got.dtype == out
    M.check_product(got, xq, wq, bias, "values")
    kept = K.mx_quantise(x)
    again = K.mx_linear(kept, weight, bias, dtype=out)
    assert torch.equal(again, got), "codes and values differ"
    plain = K.mx_linear(kept, weight, dtype=out)
    M.check_product(plain, xq, wq, None, "no bias")


# Sizes that take tiles of 128 and of 256, with one, an odd and an even number of steps of the sum.
@pytest.mark.parametrize("rows,width,outputs", [
    (2300, 200, 1100), (2301, 700, 1129), (2304, 1024, 1152), (1999, 1793, 1283), (8193, 256, 1030),
    (8200, 513, 1001), (4099, 1000, 2111), (12288, 2048, 1024), (16400, 1155, 999), (70, 2100, 70000),
    (50001, 300, 2048)])
@pytest.mark.parametrize("out", [BF, FP, F32], ids=str)
def test_large_products(cuda, rows, width, outputs, out):
    print(f"case {rows} {width} {outputs}", flush=True)
    x = make(20, rows, width, dtype=out, spread=0.5)
    weight = K.mx_quantise(make(21, outputs, width, dtype=F32, spread=0.5) / width ** 0.5)
    bias, kept = make(22, outputs, dtype=out), K.mx_quantise(x)
    got = K.mx_linear(kept, weight, bias, dtype=out)
    values = [K.mx_dequantise(m, F32).double() for m in (kept, weight)]
    for first in range(0, rows, 4096):
        part = slice(first, first + 4096)
        M.check_product(got[part], values[0][part], values[1], bias, f"rows from {first}")
    assert torch.equal(K.mx_linear(x, weight, bias), got)
    # in place of another tensor's columns, whose neighbours stay
    frame = torch.full((rows, outputs + 21), 5.0, dtype=out, device="cuda")
    K.mx_linear(kept, weight, bias, dtype=out, out=frame[:, 11:11 + outputs])
    assert torch.equal(frame[:, 11:11 + outputs], got)
    assert (frame[:, :11] == 5).all() and (frame[:, 11 + outputs:] == 5).all()


@pytest.mark.parametrize("rows,width,outputs", [(1, 512, 512), (40, 300, 90), (300, 512, 300)])
def test_products_of_scales(cuda, rows, width, outputs):
    """Blocks far apart in size, and NaN rows that stay in their row or column."""
    x, w = make(8, rows, width, dtype=F32), make(9, outputs, width, dtype=F32)
    g = torch.Generator().manual_seed(1)
    for t in (x, w):
        power = torch.randint(-20, 20, (t.shape[0], -(-width // 32)), generator=g).cuda()
        t.mul_(torch.exp2(power.float()).repeat_interleave(32, 1)[:, :width])
    x[0, width - 1] = float("inf")
    w[outputs // 2, 3] = float("nan")
    weight = K.mx_quantise(w)
    M.check_product(K.mx_linear(x, weight, dtype=F32), M.rounded(x, "fp4"), M.read(weight), None, "nan")


@pytest.mark.parametrize("rows", [1, 3, 50, 300])
def test_product_views(cuda, rows):
    """Leading dimensions, slices as rows, and results as slices with what lies beside them kept."""
    wide = make(10, 2, rows, 900)
    weight, bias = K.mx_quantise(make(11, 200, 300, dtype=F32)), make(12, 400)[::2]
    for x in (wide[..., 1:301], wide[..., 600:], wide[:, :1, :300].expand(2, rows, 300)):
        want = K.mx_linear(x.contiguous(), weight, bias.contiguous())
        assert want.shape == (2, rows, 200)
        assert torch.equal(K.mx_linear(x, weight, bias), want)
        for dtype in (BF, F32):
            frame = torch.full((2, rows, 611), 3.0, dtype=dtype, device="cuda")
            out = frame[..., 205:405]
            assert K.mx_linear(x, weight, bias, dtype=dtype, out=out) is out
            assert torch.equal(out, K.mx_linear(x, weight, bias, dtype=dtype))
            assert (frame[..., :205] == 3).all() and (frame[..., 405:] == 3).all()
    assert K.mx_linear(wide[:, :0, :300], weight).shape == (2, 0, 200)
    assert K.mx_linear(wide[0, 0, :300], weight).shape == (200,)


def test_streams_and_graphs(cuda):
    """A call on another stream, and a captured chain replayed on new inputs between eager work."""
    x, weight = make(13, 300, 520), K.mx_quantise(make(14, 130, 520, dtype=F32))
    few = x[:3].clone()
    want = [K.mx_linear(x, weight), K.mx_linear(few, weight), K.mx_dequantise(K.mx_quantise(x, "int8"))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [K.mx_linear(x, weight), K.mx_linear(few, weight),
               K.mx_dequantise(K.mx_quantise(x, "int8"))]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [K.mx_linear(x, weight), K.mx_linear(few, weight),
               K.mx_dequantise(K.mx_quantise(x, "int8"))]
    for seed in (15, 16, 17):
        x.copy_(make(seed, 300, 520))
        few.copy_(x[:3])
        graph.replay()
        torch.cuda.synchronize()
        want = [K.mx_linear(x, weight), K.mx_linear(few, weight),
                K.mx_dequantise(K.mx_quantise(x, "int8"))]
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_far_offsets(cuda):
    """Rows whose elements lie more than 2^31 apart from the first, in and out."""
    rows, width = 70000, 31
    base = torch.zeros(rows * 40000 if torch.cuda.mem_get_info()[0] > 20 << 30 else 0, dtype=BF,
                       device="cuda")
    if base.numel() == 0:
        pytest.skip("needs 6 GB")
    x = base.view(rows, 40000)[:, 3:3 + width]
    fill = make(18, rows, width)
    x.copy_(fill)
    m, want = K.mx_quantise(x, "int8"), K.mx_quantise(fill, "int8")
    assert torch.equal(m.codes, want.codes) and torch.equal(m.scales, want.scales)
    x.zero_()
    K.mx_dequantise(m, BF, out=x)
    assert torch.equal(x, K.mx_dequantise(want))
    weight = K.mx_quantise(make(19, 17, width, dtype=F32))
    out = base.view(rows, 40000)[:, 100:117]
    assert torch.equal(K.mx_linear(fill, weight, out=out), K.mx_linear(fill, weight))

"""Host checks of the microscaled forms: their refusals (before any launch; the pointers given to the
C entry points are never dereferenced), the layouts they allocate, and the tests' own 64-bit form
against the formats' properties."""

import pytest
import torch

import mx_util as M
from recap_amd import _lib
from recap_amd import kernels as K

BF, F32 = torch.bfloat16, torch.float32
X = torch.zeros(4, 6, 96, dtype=BF)
W = K.Microscaled.empty((40, 96), "fp4")
X4 = K.Microscaled.empty((4, 6, 96), "fp4")
I8 = K.Microscaled.empty((40, 96), "int8")


@pytest.mark.parametrize("format,width,row,scales", [
    ("fp4", 1, 128, 8), ("fp4", 256, 128, 8), ("fp4", 257, 256, 16), ("int8", 1, 32, 1),
    ("int8", 32, 32, 1), ("int8", 128, 128, 4), ("int8", 129, 160, 5)])
def test_layouts(format, width, row, scales):
    m = K.Microscaled.empty((3, 2, width), format)
    assert m.codes.shape == (3, 2, row) and m.scales.shape == (3, 2, scales)
    assert m.shape == (3, 2, width) and m.nbytes() == 6 * (row + scales)
    code = {"fp4": _lib.MX_FP4, "int8": _lib.MX_INT8}[format]
    lib = _lib.load()
    assert lib.recap_mx_row_bytes(code, width) == row
    assert lib.recap_mx_row_scales(code, width) == scales
    assert lib.recap_mx_row_bytes(3, width) == lib.recap_mx_row_scales(code, 0) == -1


def test_workspace_size():
    size = _lib.load().recap_mx_linear_workspace_size
    assert size(100, 300, 7, 0) == 100 * (256 + 16) and size(100, 300, 7, 1) == 0
    assert size(5, 300, 7, 0) == 0      # few rows: brought into fp4 where they are multiplied
    assert size(0, 300, 7, 0) == size(5, 0, 7, 0) == size(5, 300, 0, 1) == -1
    assert size(5, (1 << 22) + 1, 7, 0) == size((1 << 29) + 1, 300, 7, 0) == -1
    assert size(5, 300, (1 << 29) + 1, 1) == size(1 << 20, 300, (1 << 17) + 1, 1) == -1


def wide_out(strides, dtype=BF, shape=(4, 6, 40)):
    return torch.empty_strided(shape, strides, dtype=dtype)


@pytest.mark.parametrize("call,match", [
    (lambda: K.mx_quantise(X, "fp8"), "format"),
    (lambda: K.mx_quantise(X.double()), "dtype"),
    (lambda: K.mx_quantise(torch.zeros((), dtype=BF)), "width"),
    (lambda: K.mx_quantise(torch.zeros(3, 0, dtype=BF)), "width"),
    (lambda: K.mx_quantise(X), "GPU"),
    (lambda: K.mx_quantise(X, "fp4", out=I8), "int8"),
    (lambda: K.mx_quantise(X, "fp4", out=W), "microscaled form"),
    (lambda: K.mx_quantise(X[..., :64], "fp4", out=X4), "microscaled form"),
    (lambda: K.Microscaled.empty((3, 0), "fp4"), "rows of 0"),
    (lambda: K.Microscaled.empty((3, 32), "int4"), "format"),
    (lambda: K.mx_dequantise(X4, torch.float64), "dtype"),
    (lambda: K.mx_dequantise(X4, torch.int8), "dtype"),
    (lambda: K.mx_dequantise(X4), "GPU"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales, "fp8", 96)), "format"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales, "int8", 96)), "codes"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales, "fp4", 300)), "codes"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales, "fp4", 0)), "rows of 0"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales[:3], "fp4", 96)), "scales"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes, X4.scales.float(), "fp4", 96)), "scales"),
    (lambda: K.mx_dequantise(K.Microscaled(X4.codes.transpose(0, 1), X4.scales.transpose(0, 1),
                                           "fp4", 96)), "contiguous"),
    (lambda: K.mx_linear(X, I8), "int8"),
    (lambda: K.mx_linear(K.Microscaled.empty((4, 96), "int8"), W), "int8"),
    (lambda: K.mx_linear(X, X4), "outputs, width"),
    (lambda: K.mx_linear(X[..., :95], W), "takes rows of 96"),
    (lambda: K.mx_linear(K.Microscaled.empty((4, 95), "fp4"), W), "takes rows of 96"),
    (lambda: K.mx_linear(X.double(), W), "dtype"),
    (lambda: K.mx_linear(torch.zeros((), dtype=BF), W), "width"),
    (lambda: K.mx_linear(X, W, dtype=torch.float64), "dtype"),
    (lambda: K.mx_linear(X, W, torch.zeros(39)), "bias"),
    (lambda: K.mx_linear(X, W, torch.zeros(1, 40)), "bias"),
    (lambda: K.mx_linear(X, W, torch.zeros(40, dtype=torch.float64)), "bias"),
    (lambda: K.mx_linear(X, W), "GPU"),
    (lambda: K.mx_linear(X4, W), "GPU"),
    (lambda: K.mx_linear(X, K.Microscaled(W.codes[:39], W.scales, "fp4", 96)), "scales"),
    (lambda: K.mx_linear(X.clone().requires_grad_(), W), "gradient"),
    (lambda: K.mx_linear(X, W, torch.zeros(40, requires_grad=True)), "gradient"),
    (lambda: K.mx_quantise(X.clone().requires_grad_()), "gradient")])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def c_call(name, **change):
    """An entry point's call with sound arguments but for those in `change`."""
    base = dict(
        recap_mx_quantise=dict(values=64, dtype=2, rows=4, width=96, stride=96, format=1, codes=64,
                               scales=64, stream=None),
        recap_mx_dequantise=dict(codes=64, scales=64, format=1, rows=4, width=96, values=64, dtype=2,
                                 stride=96, stream=None),
        recap_mx_linear=dict(x=64, x_dtype=2, x_stride=96, x_scales=None, rows=40, width=96, w=64,
                             w_scales=64, outputs=40, bias=64, bias_dtype=2, out=64, dtype=2,
                             out_stride=40, work=64, work_bytes=40 * 136, stream=None))[name]
    assert set(change) <= set(base)
    return _lib.call(name, *{**base, **change}.values())


@pytest.mark.parametrize("name,change", [
    *(("recap_mx_quantise", c) for c in (
        dict(values=None), dict(codes=None), dict(scales=None), dict(dtype=4), dict(format=0),
        dict(format=3), dict(rows=0), dict(width=0), dict(width=(1 << 24) + 1), dict(rows=1 << 31),
        dict(stride=-1), dict(values=65), dict(values=66, dtype=3), dict(codes=72))),
    *(("recap_mx_dequantise", c) for c in (
        dict(values=None), dict(codes=None), dict(scales=None), dict(dtype=0), dict(format=7),
        dict(rows=-1), dict(width=0), dict(stride=95), dict(stride=0), dict(values=65), dict(codes=72))),
    *(("recap_mx_linear", c) for c in (
        dict(x=None), dict(w=None), dict(w_scales=None), dict(out=None), dict(work=None),
        dict(work_bytes=40 * 136 - 1), dict(work=72), dict(x_dtype=5), dict(dtype=4), dict(bias_dtype=9),
        dict(rows=0), dict(width=0), dict(outputs=0), dict(width=(1 << 22) + 1), dict(outputs=1 << 31),
        dict(rows=(1 << 29) + 1, x_scales=64), dict(rows=1 << 20, outputs=(1 << 17) + 1, x_scales=64),
        dict(x_stride=-96), dict(x=65), dict(out=65), dict(out=66, dtype=3), dict(bias=65),
        dict(bias=66, bias_dtype=3), dict(out_stride=39), dict(w=72), dict(w_scales=68),
        dict(x_scales=68), dict(x=72, x_scales=64)))])
def test_c_refusals(name, change):
    """Each is turned down on the host: no GPU is there to be reached."""
    with pytest.raises(ValueError, match=name[6:]):
        c_call(name, **change)


@pytest.mark.parametrize("format", ["fp4", "int8"])
def test_the_definition(format):
    """Half a step at most, of the value's own binade (fp4) or of the block's (int8); what is on the
    grid stays; a block keeps its scale under its own rounding."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(200, 100, generator=g, dtype=torch.float64) * torch.randn(100, generator=g).exp()
    index, negative, byte = M.quantise(x, format)
    got = M.values(index, negative, byte, format, 100)
    unit = (2.0 ** (byte.double() - 127)).repeat_interleave(32, 1)[:, :100]
    step = unit / 64 if format == "int8" else torch.maximum(
        unit / 2, 2.0 ** torch.floor(torch.log2(x.abs().clamp_min(1e-30))) / 2)
    assert ((got - x).abs() <= step / 2 * (1 + 1e-12)).all()
    again = M.quantise(got, format)
    assert torch.equal(M.values(*again, format, 100), got)
    codes = M.pack(index, negative, format)
    assert all(torch.equal(a, b) for a, b in zip(M.unpack(codes, format), (
        index, negative if format == "fp4" else negative & (index > 0))))


@pytest.mark.parametrize("name,args,match", [
    ("recap_refresh_capture_mx", [64, 2, 1, 2, 64, 64, 64, 64, *[64] * 6, 256, 256, 64, None, 64,
                                  *[None] * 5], "det_scale is NULL"),
    ("recap_refresh_capture_mx", [64, 2, 1, 2, 64, 64, 64, 64, *[64] * 6, 256, 256, 72, 64, 64,
                                  *[None] * 5], "alignment"),
    ("recap_sparse_merge_attn_mx", [64, 2, 1, 2, 64, 64, 64, 64, *[64] * 4, 256, 256, 0.125, 64, 64,
                                    64, None, 64, 64, 64, -1.0, 64, 64, 64, 64, 1, 1, 64, 1 << 30,
                                    None], "det_scale is NULL"),
    ("recap_sparse_merge_attn_mx", [64, 2, 1, 2, 64, 64, 64, 64, *[64] * 4, 256, 256, 0.125, 64, 64,
                                    64, 66, 64, 64, 64, -1.0, 64, 64, 64, 64, 1, 1, 64, 1 << 30,
                                    None], "4-byte aligned"),
    ("recap_sparse_call_mx", [64, 64, 64, 2, 1, 2, 64, *[64] * 9, 64, 256, 256, 0.125, 2.0, 4, 8, 1,
                              *[64] * 6, None, 64, 64, -1.0, 64, 64, 64, 64, 1, None, 64, 1 << 30,
                              None], "det_scale is NULL")])
def test_c_refinement_refusals(name, args, match):
    with pytest.raises(ValueError, match=match):
        _lib.call(name, *args)


def test_bank_format_is_checked():
    from recap_amd import HostBankOperator, Operator, OperatorConfig
    from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation

    geometry = SparseGeometry.build(Layout.from_permutation(hilbert_permutation((2, 8, 16)),
                                                            text_tokens=0, text_first=False), 128)
    for cls in (Operator, HostBankOperator):
        assert cls.build(OperatorConfig(), geometry, n_layers=1).bank_format == "fp16"
        assert cls.build(OperatorConfig(), geometry, n_layers=1, bank_format="int8").bank_format == "int8"
        with pytest.raises(ValueError, match="bank_format"):
            cls.build(OperatorConfig(), geometry, n_layers=1, bank_format="fp4")

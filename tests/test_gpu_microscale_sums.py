"""The fp32 sums of mx_linear on the GPU, bit for bit: operands whose sums fp32 holds exactly in any
order, over every kernel's sizes and number of steps, and a bias far larger than the products."""

import pytest
import torch

import mx_sums as S
from recap_amd import kernels as K

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32

# A few rows, then tiles of 64, of 128 and of 256: one step of the sum to many, odd and even.
SIZES = [(1, 31, 1), (2, 256, 40), (1, 8192, 2000), (7, 20001, 65), (8, 8192, 70), (8, 1300, 10300),
         (16, 3841, 32), (16, 4096, 33), (16, 8192, 40),
         (9, 300, 33), (9, 2500, 65), (17, 4096, 31), (33, 8192, 64), (64, 20001, 65), (200, 2048, 96),
         (2300, 200, 1100), (2301, 1793, 1129), (4099, 1000, 2111), (8200, 2500, 1030), (12288, 2048, 1024)]


def operands(rows, width, outputs):
    g = torch.Generator().manual_seed(rows + width + outputs)
    return S.operand(g, rows, width).cuda(), S.operand(g, outputs, width).cuda()


@pytest.mark.parametrize("rows,width,outputs", SIZES)
def test_sums_are_exact(cuda, rows, width, outputs):
    print(f"case {rows} {width} {outputs}", flush=True)
    x, w = operands(rows, width, outputs)
    weight, kept = K.mx_quantise(w), K.mx_quantise(x)
    assert torch.equal(K.mx_dequantise(weight, F32), w) and torch.equal(K.mx_dequantise(kept, F32), x)
    for out in (F32, BF, FP):
        S.check_exact(K.mx_linear(kept, weight, dtype=out), x, w, None, f"{out}")
    S.check_exact(K.mx_linear(x, weight, dtype=F32), x, w, None, "values")

@pytest.mark.parametrize("rows,width,outputs", SIZES)
def test_large_bias(cuda, rows, width, outputs):
    """The bias is added to the whole sum, with one rounding: 1e4 and more times the products, it takes
    nothing from them but that."""
    print(f"case {rows} {width} {outputs}", flush=True)
    x, w = operands(rows, width, outputs)
    weight = K.mx_quantise(w)
    g = torch.Generator(device="cuda").manual_seed(width)
    for size in (1e4, 1e8):
        bias = size * torch.randn(outputs, generator=g, device="cuda")
        for out in (F32, BF):
            S.check_exact(K.mx_linear(x, weight, bias, dtype=out), x, w, bias, f"{size} {out}")
    few = K.mx_linear(x[:1], weight, bias, dtype=F32)
    assert torch.equal(few, K.mx_linear(x, weight, bias, dtype=F32)[:1])

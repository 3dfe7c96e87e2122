"""The test of an fp4 product's sum, tested itself: it accepts fp32 sums in every order and rejects
what its sizes must not hide, a block of 32 left out and partial sums in 16 bits."""

import pytest
import torch

import mx_sums as S
import mx_util as M

F32 = torch.float32


def operands(rows, width, outputs):
    g = torch.Generator().manual_seed(rows + width + outputs)
    return S.operand(g, rows, width), S.operand(g, outputs, width)


def summed(x, w, step, dtype):
    """The product with its sum kept in `dtype` after every `step` values."""
    total = torch.zeros(x.shape[0], w.shape[0], dtype=dtype)
    for first in range(0, x.shape[1], step):
        part = slice(first, first + step)
        total = (total.double() + x[:, part].double() @ w[:, part].double().T).to(dtype)
    return total.float()


@pytest.mark.parametrize("width", [31, 300, 4096])
def test_operands_are_their_own_form(width):
    x = operands(5, width, 1)[0]
    assert torch.equal(M.rounded(x, "fp4"), x.double())


@pytest.mark.parametrize("width", [1, 300, 5000, 20001])
def test_accepts_every_order(width):
    x, w = operands(7, width, 33)
    order = torch.randperm(width, generator=torch.Generator().manual_seed(1))
    for a, b in ((x, w), (x[:, order], w[:, order])):
        S.check_exact(summed(a, b, 64, F32), x, w, None, "in turn")
    halves = [summed(x[:, i::8], w[:, i::8], 64, F32) for i in range(8)]
    S.check_exact(sum(halves), x, w, None, "in eight parts")
    S.check_exact(sum(halves).bfloat16(), x, w, None, "rounded once")


@pytest.mark.parametrize("width", [512, 3841, 4096, 8192, 20001])
def test_rejects_what_is_wrong(width):
    x, w = operands(7, width, 33)
    right = summed(x, w, 64, F32)
    for block in (0, width // 64, -(-width // 32) - 1):
        part = slice(32 * block, 32 * block + 32)
        with pytest.raises(AssertionError, match="differ"):
            S.check_exact(right - (x[:, part] @ w[:, part].T), x, w, None, "a block less")
    for step, dtype in ((64, torch.float16), (256, torch.bfloat16)):
        with pytest.raises(AssertionError, match="differ"):
            S.check_exact(summed(x, w, step, dtype), x, w, None, "16-bit sums")
    bias = torch.full((33,), 1.0e8) + 1000 * torch.arange(33)
    S.check_exact((right.double() + bias.double()).float(), x, w, bias, "the bias last")
    total = bias.expand(7, 33)
    for first in range(0, width, 64):
        total = total + x[:, first:first + 64] @ w[:, first:first + 64].T
    with pytest.raises(AssertionError, match="differ"):
        S.check_exact(total, x, w, bias, "the bias first")


def test_refuses_operands_that_need_more_bits():
    x = torch.full((1, 1 << 20), 24.0)
    with pytest.raises(AssertionError, match="24 bits"):
        S.check_exact(torch.zeros(1, 1), x, x, None, "too long")

"""The microscaled forms together, as a served model uses them: an attention block whose projections
are in fp4 over an operator whose banks are in int8, refresh then sparse steps."""

import pytest
import torch

import recap_amd
from gpu_util import SMALL
from recap_amd import REFRESH, SPARSE, OperatorConfig, kernels as K
from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation

pytestmark = pytest.mark.gpu


def build(wl, cls, width=320, seed=0):
    layout = Layout.from_permutation(hilbert_permutation(wl.grid), text_tokens=wl.text_tokens,
                                     text_first=wl.text_first)
    op = cls.build(OperatorConfig(head_density=wl.density, host_banks=cls is recap_amd.HostBankOperator),
                   SparseGeometry.build(layout, 128), n_layers=1, bank_format="int8")
    torch.manual_seed(seed)
    inner = wl.heads * wl.dim
    layers = {n: torch.nn.Linear(*s, device="cuda", dtype=wl.dtype)
              for n, s in (("q", (width, inner)), ("k", (width, inner)), ("v", (width, inner)),
                           ("o", (inner, width)))}
    micro = {n: recap_amd.MicroscaledLinear.from_linear(m) for n, m in layers.items()}
    block = recap_amd.AttentionBlock(op, 0, wl.heads, micro["q"], micro["k"], micro["v"], micro["o"],
                                     dtype=wl.dtype, norm="rms", next_norm="rms")
    return block, micro, layers


@pytest.mark.parametrize("name,stream", [("text-last-d128", torch.float32),
                                         ("text-first-ragged", torch.bfloat16)])
def test_steps(cuda, name, stream):
    """The block against its parts one by one, bit for bit, resident and paged."""
    wl = SMALL[name]
    block, micro, _ = build(wl, recap_amd.Operator)
    paged, _, _ = build(wl, recap_amd.HostBankOperator)
    ref, _, _ = build(wl, recap_amd.Operator)
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    scale, shift, gate = (0.3 * rand(1, 1, 320) for _ in range(3))
    x = rand(1, wl.tokens, 320).to(stream)
    for step, kind in enumerate((REFRESH, SPARSE, SPARSE)):
        for b in (block, paged, ref):
            b.operator.begin_step(step, kind)
        r, y = block(x, scale, shift, gate)
        r2, y2 = paged(x, scale, shift, gate)
        assert torch.equal(r, r2) and torch.equal(y, y2)
        h = K.norm_modulate(x, scale, shift, norm="rms", dtype=wl.dtype)
        q, k, v = (K.mx_linear(h, micro[n].weight, micro[n].bias).unflatten(2, (wl.heads, wl.dim))
                   .transpose(1, 2) for n in "qkv")
        out = ref.operator.attend(0, *K.qk_rotary(q, k), v)
        branch = K.mx_linear(out.transpose(1, 2).flatten(2), micro["o"].weight, micro["o"].bias)
        want = K.gated_residual_norm(x, branch, gate, norm="rms")
        assert torch.equal(r, want[0]) and torch.equal(y, want[1])
        assert torch.isfinite(r).all()
        x = (x + 0.02 * rand(1, wl.tokens, 320)).to(stream)


def test_linear_layer(cuda):
    """A torch layer's form: its weight as it was, one call for values and for codes, its dtype."""
    torch.manual_seed(2)
    layer = torch.nn.Linear(300, 130, device="cuda", dtype=torch.bfloat16)
    micro = recap_amd.MicroscaledLinear.from_linear(layer)
    x = torch.randn(2, 7, 300, device="cuda", dtype=torch.bfloat16)
    want = K.mx_linear(x, K.mx_quantise(layer.weight.detach()), layer.bias.detach())
    assert want.dtype == torch.bfloat16 and want.shape == (2, 7, 130)
    assert torch.equal(micro(x), want) and torch.equal(micro(K.mx_quantise(x)), want)
    with torch.no_grad():
        layer.weight.zero_()
        layer.bias.zero_()
    assert torch.equal(micro(x), want)
    wide = recap_amd.MicroscaledLinear(micro.weight, dtype=torch.float32)
    assert wide(x).dtype == torch.float32 and micro(x, dtype=torch.float16).dtype == torch.float16
    # against the product of the unrounded x: its values are off by up to a fifth, or 1/14 of the block
    plain = torch.nn.functional.linear(x.float(), K.mx_dequantise(micro.weight, torch.float32))
    assert (wide(x) - plain).norm() < 0.25 * plain.norm()

"""The refinement bank in int8 on the GPU: captures against the definition in 64 bits, merges and
validations bit for bit against the same values held in fp16, and the operator's steps with it,
resident, in groups of heads and paged."""

import dataclasses

import pytest
import torch

import mx_util as M
from gpu_util import SMALL
from recap_amd import (HostBankOperator, Operator, OperatorConfig, REFRESH, SPARSE, kernels as K)
from recap_amd.layout import Layout, SparseGeometry, hilbert_permutation
from recap_amd.synthetic import make_qkv, perturb

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def parts(seed, batch, heads, dim, n_video, n_text, dtype=BF, spread=1.0):
    """A capture's inputs: dense and head branch with their masses, the coarse tail, a row order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    n, banks, rows = n_video + n_text, batch * heads, n_video // 128 * 128
    rowmap = torch.cat([torch.randperm(n_video, generator=g, device="cuda"),
                        torch.arange(n_video, n, device="cuda")]).int()
    lse = 5 + rand(banks, n)
    ratio = torch.rand(banks, n, generator=g, device="cuda")
    ratio[:, ::7] = 1 - 10 ** (-1 - 7 * torch.rand(banks, len(ratio[0, ::7]), generator=g, device="cuda"))
    dense_lse = torch.empty_like(lse)
    dense_lse[:, rowmap.long()] = lse
    size = (spread * rand(dim)).exp()
    far = torch.zeros(rows, device="cuda")      # masses past their limits of +-30
    far[3::11], far[8::11] = 1, -1
    return dict(dense_out=(rand(batch, heads, n, dim) * size).to(dtype),
                dense_lse=dense_lse.view(batch, heads, n), head_out=(rand(banks, n, dim) * size).to(dtype),
                head_lse=lse + ratio.log(), go=(rand(banks, rows, dim) * size).to(dtype),
                gl=4 + rand(banks, rows) + 60 * far, rowmap=rowmap, geo=K.Geometry(n, n_video))


def empty_bank(p):
    banks, rows, dim = p["go"].shape
    return (K.Microscaled.empty((banks, rows, dim), "int8", "cuda"),
            torch.zeros(banks, rows, device="cuda"))


def detail(p):
    """((value, bound of its fp32 arithmetic), (mass, its bound)) in 64 bits, before the codes."""
    rows, dim = p["go"].shape[1:]
    at = p["rowmap"][:rows].long()
    of = p["dense_out"].flatten(0, 1)[:, at].double()
    lf = p["dense_lse"].flatten(0, 1)[:, at].double()
    oh, lh = p["head_out"][:, :rows].double(), p["head_lse"][:, :rows].double()
    go, gl = p["go"].double(), p["gl"].double()
    less = (lh - lf).clamp(max=0)
    ratio = less.exp().clamp(max=1 - 1e-6)
    rest = (-torch.expm1(less)).clamp(min=1e-6)
    r, q = ratio[..., None], rest[..., None]
    value = ((of - r * oh) / q - go).clamp(-6e4, 6e4)
    # fp32: lh - lf is exact here within its own rounding (2^-24 of the masses' size, which moves
    # ratio by as much and rest by that over itself); eight more roundings of 2^-24 each.
    e = 2.0 ** -24
    near = (lh - lf).abs() * e
    bound = ((of.abs() + (r * oh).abs()) / q * (8 * e + (near / rest)[..., None])
             + go.abs() * 2 * e + value.abs() * 4 * e + (near[..., None] * (r * oh).abs()) / q)
    mass = lf + torch.log(rest) - gl
    mass_bound = near / rest + 8 * e * (1 + (lf - gl).abs() + torch.log(rest).abs() + mass.abs())
    border = (ratio - (1 - 1e-3)).abs() < 1e-6
    zero = (ratio > 1 - 1e-3)[..., None]
    return (torch.where(zero, 0.0, value), torch.where(zero, 0.0, bound), border), (mass.clamp(-30, 30), mass_bound)


@pytest.mark.parametrize("batch,heads,dim,n_video,n_text,dtype", [
    (1, 2, 64, 256, 0, BF), (2, 3, 128, 500, 77, BF), (1, 1, 128, 128, 1, FP), (1, 5, 64, 1031, 30, FP)])
def test_capture(cuda, batch, heads, dim, n_video, n_text, dtype):
    p = parts(1, batch, heads, dim, n_video, n_text, dtype)
    bank, mass = empty_bank(p)
    print(f"case {batch} {heads} {dim} {n_video} {n_text}", flush=True)
    assert K.refresh_capture(*p.values(), bank, mass) is None
    (value, bound, border), (want_mass, mass_bound) = detail(p)
    got = M.read(bank)
    value, bound, keep = value.cpu(), bound.cpu(), ~border.cpu()
    # each value within half a step of its block as the capture scaled it, and the arithmetic
    step = (2.0 ** (bank.scales.cpu().double() - 133)).repeat_interleave(32, -1)
    off = ((got - value).abs() / (step / 2 + bound))[keep]
    assert off.max() <= 1, off.max()
    # and that scale is the definition's, but for blocks whose largest value is within the bound
    # of a border
    low, high = (M.quantise(v, "int8")[2] for v in ((value.abs() - bound).clamp(min=0),
                                                    value.abs() + bound))
    scales = bank.scales.cpu()
    ok = (scales == low) | (scales == high)
    assert ok[keep[..., None].expand_as(ok)].all()
    assert (low == high).double().mean() > 0.9
    off = ((mass.double() - want_mass).abs() / mass_bound).cpu()[keep]
    assert off.max() <= 1, off.max()


@pytest.mark.parametrize("batch,heads,dim,n_video,n_text", [(1, 2, 64, 256, 0), (2, 3, 128, 500, 77)])
def test_validation(cuda, batch, heads, dim, n_video, n_text):
    """A validating capture scores what the bank held before, as one of fp16 with the same values."""
    p, q = (parts(s, batch, heads, dim, n_video, n_text) for s in (2, 3))
    bank, mass = empty_bank(p)
    K.refresh_capture(*p.values(), bank, mass)
    half, half_mass = K.mx_dequantise(bank, FP), mass.clone()
    assert torch.equal(half.double().cpu(), M.read(bank))  # these values are fp16's too
    center = torch.randn(batch * heads, device="cuda")
    got = K.refresh_capture(*q.values(), bank, mass, glref=p["gl"], center=center)
    want = K.refresh_capture(*q.values(), half, half_mass, glref=p["gl"], center=center)
    assert torch.equal(got, want)
    fresh, fresh_mass = empty_bank(q)
    K.refresh_capture(*q.values(), fresh, fresh_mass)
    assert torch.equal(bank.codes, fresh.codes) and torch.equal(bank.scales, fresh.scales)
    assert torch.equal(mass, fresh_mass)


def test_capture_limits(cuda):
    """Values past 6e4 are kept as what 6e4 rounds to, rows whose head holds all of the mass as 0."""
    p = parts(5, 1, 1, 64, 128, 0)
    p["dense_lse"].fill_(2.0)
    p["head_lse"].fill_(2.0 - 0.6931472)    # half of the mass
    p["head_lse"][:, 64:] = 3.0             # more than all
    p["dense_out"].fill_(1.0e5)
    p["dense_out"][..., 32:] *= -1
    p["head_out"].zero_()
    p["go"].zero_()
    bank, mass = empty_bank(p)
    K.refresh_capture(*p.values(), bank, mass)
    got = M.read(bank)
    assert (got[:, :64, :32] == 59904).all() and (got[:, :64, 32:] == -59904).all()
    assert (got[:, 64:] == 0).all()


def build(cls, wl, chunks=1, layers=1, streams=1, **more):
    layout = Layout.from_permutation(hilbert_permutation(wl.grid), text_tokens=wl.text_tokens,
                                     text_first=wl.text_first)
    cfg = OperatorConfig(head_density=wl.density, bank_chunks=chunks)
    if cls is HostBankOperator:
        cfg = dataclasses.replace(cfg, host_banks=True)
    return cls.build(cfg, SparseGeometry.build(layout, 128), n_layers=layers, n_streams=streams, **more)


def inputs(wl, steps, device, seed=0):
    first = make_qkv(wl, seed=seed)
    return [tuple((x if s == 0 else perturb(x, 0.02, seed=seed, step=s)).to(device) for x in first)
            for s in range(steps)]


@pytest.mark.parametrize("name", list(SMALL))
@pytest.mark.parametrize("alpha", [None, 0.0, 0.4])
def test_merge_reads_the_values(cuda, name, alpha):
    """Sparse calls with the int8 bank, and with its values in an fp16 bank: the same bits; both of
    the one library call and of the separate stages."""
    wl = SMALL[name]
    (q0, k0, v0), (q1, k1, v1) = inputs(wl, 2, cuda)
    ops = [build(Operator, wl, bank_format="int8"), build(Operator, wl)]
    outs = []
    for op in ops:
        op.begin_step(0, REFRESH)
        outs.append(op.attend(0, q0, k0, v0))
        op.alpha_override = alpha
    assert torch.equal(*outs)
    small, full = (op.banks[0][0] for op in ops)
    assert small.value.dtype == torch.int8 and full.value_scale is None
    rows, d = small.value.shape[1:]
    assert small.refinement_bytes() == small.value.shape[0] * rows * (d + d // 32 + 4)
    assert full.refinement_bytes() == small.value.shape[0] * rows * (2 * d + 4)
    full.value, full.log_mass = K.mx_dequantise(small.refinement(), FP), small.log_mass.clone()
    assert torch.equal(full.value.double().cpu(), M.read(small.refinement()))
    outs = []
    for op in ops:
        op.begin_step(1, SPARSE)
        outs.append(op.attend(0, q1, k1, v1))
    assert torch.equal(*outs)
    staged = []
    for op in ops:
        op.layers[0][0].reset()      # a bank that was handed in: no basis yet
        op.begin_step(2, SPARSE)
        staged.append(op.attend(0, q1, k1, v1))
    assert torch.equal(*staged)


@pytest.mark.parametrize("name", ["text-last-d128", "text-first-ragged"])
def test_steps(cuda, name):
    """Two layers and streams, a refresh, sparse steps and a validating refresh: resident, in groups
    of heads and paged all alike, the error measure near the fp16 bank's."""
    wl = SMALL[name]
    ops = [build(cls, wl, chunks, layers=2, streams=2, bank_format="int8")
           for cls, chunks in ((Operator, 1), (Operator, 2), (HostBankOperator, 1), (HostBankOperator, 3))]
    ops.append(build(Operator, wl, layers=2, streams=2))
    steps = {(s, l): inputs(wl, 5, cuda, seed=10 * s + l) for s in range(2) for l in range(2)}
    for step, kind in enumerate((REFRESH, SPARSE, SPARSE, REFRESH, SPARSE)):
        for op in ops:
            op.begin_step(step, kind)
        for (stream, layer), calls in steps.items():
            outs = []
            for op in ops:
                op.set_stream(stream)
                outs.append(op.attend(layer, *calls[step]))
            for other in outs[1:-1]:
                assert torch.equal(outs[0], other), (step, stream, layer)
            # the fp16 bank's output: what a step of the refinement and the rounding can move
            assert (outs[0].double() - outs[-1].double()).abs().max() < 0.05
        errors = [op.drain_validation() for op in ops]
        if step == 3:
            ages, values = zip(*errors)
            assert set(ages) == {3}
            assert max(values[:-1]) - min(values[:-1]) <= 1e-6 * values[0]  # sums in another order
            assert abs(values[-1] - values[0]) < 0.02 * values[-1]
    resident, paged = ops[0], ops[2]
    banks, rows, d = wl.heads, resident.banks[0][0].log_mass.shape[1], wl.dim
    assert resident.peak_bank_bytes() == 4 * banks * rows * (d + d // 32 + 4)
    assert paged.peak_bank_bytes() < ops[-1].peak_bank_bytes() + 4 * sum(
        t.numel() * t.element_size() for t in (resident.banks[0][0].partition,
                                               resident.banks[0][0].head_kernel_mask,
                                               resident.banks[0][0].coarse_lse))
    assert set(paged._slots[0]) == {"value", "log_mass", "partition", "head_kernel_mask", "coarse_lse",
                                    "value_scale"}


def test_video_under_one_block(cuda):
    """No refined rows: empty banks in both formats, the head alone."""
    wl = dataclasses.replace(SMALL["tiny"], grid=(1, 8, 12), text_tokens=200)
    calls = inputs(wl, 2, cuda)
    outs = []
    for cls, more in ((Operator, {}), (Operator, dict(bank_format="int8")),
                      (HostBankOperator, dict(bank_format="int8"))):
        op = build(cls, wl, **more)
        op.begin_step(0, REFRESH)
        first = op.attend(0, *calls[0])
        op.begin_step(1, SPARSE)
        outs.append((first, op.attend(0, *calls[1])))
    for other in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(outs[0], other))


def test_refusals(cuda):
    p = parts(4, 1, 2, 64, 256, 0)
    bank, mass = empty_bank(p)
    for bad, match in ((K.Microscaled.empty((2, 256, 64), "fp4", "cuda"), "int8 rows"),
                       (K.Microscaled.empty((2, 128, 64), "int8", "cuda"), "rows of"),
                       (K.Microscaled(bank.codes, bank.scales.cpu(), "int8", 64), "GPU"),
                       (K.Microscaled(bank.codes, bank.scales[:, :, :1], "int8", 64), "scales")):
        with pytest.raises(ValueError, match=match):
            K.refresh_capture(*p.values(), bad, mass)
    with pytest.raises(ValueError, match="refresh_capture"):
        K.refresh_capture_noalloc(*p.values(), bank, mass, None)
    with pytest.raises(ValueError, match="bank_format"):
        build(Operator, SMALL["tiny"], bank_format="int4")


def test_text_retarget_and_reset(cuda):
    """A per-prompt text length after the banks were preallocated, and a new sample: paged banks of
    another geometry, as the resident ones."""
    base = SMALL["text-last-d128"]
    wl = dataclasses.replace(base, text_tokens=16)
    resident, paged = (build(c, wl, layers=2, bank_format="int8") for c in (Operator, HostBankOperator))
    assert paged.preallocate_host(2, wl.heads, wl.dim) > 0
    for text in (16, 300, 77):
        wl = dataclasses.replace(base, text_tokens=text)
        for op in (resident, paged):
            op.reset()
            op.layout.text_tokens = text
            op.layout._gather_cache.clear()
        for step, kind in enumerate((REFRESH, SPARSE, SPARSE, REFRESH, SPARSE)):
            for layer in range(2):
                qkv = inputs(wl, step + 1, cuda, seed=layer)[step]
                outs = []
                for op in (resident, paged):
                    if layer == 0:
                        op.begin_step(step, kind)
                    outs.append(op.attend(layer, *qkv))
                assert torch.equal(*outs), (text, step, layer)


def test_graph_replays(cuda):
    """A captured sparse call with the int8 bank, replayed on new inputs between eager ones."""
    wl = SMALL["text-last-d128"]
    calls = inputs(wl, 5, cuda)
    op = build(Operator, wl, bank_format="int8")
    op.begin_step(0, REFRESH)
    op.attend(0, *calls[0])
    op.begin_step(1, SPARSE)
    held = tuple(x.clone() for x in calls[1])
    op.attend(0, *held)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = op.attend(0, *held)
    for call in calls[2:]:
        for x, new in zip(held, call):
            x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, op.attend(0, *call))
